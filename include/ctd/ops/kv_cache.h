#pragma once
// KV cache read/write ops (mirrors ops/kv_cache.h of the reference).
#include "ctd/tensor.h"

namespace ctd::ops {

// Writes src [B, T, H_kv, D] into cache [B, H_kv, max_seq, D] at rows
// [pos, pos+T), folding the axis permute into the copy.
void write_kv_inplace(Tensor& cache, const Tensor& src, int pos);

// cache[:, :, :valid_len, :] with each KV head repeated `group` times:
// [B, H_kv * group, valid_len, D].
Tensor read_kv_expanded(const Tensor& cache, int valid_len, int group);

// The same over a cache held in 4 bits (added in this build; ember_kv4_write and
// ember_kv4_read_expanded give the format): codes int32 [B, H_kv, max_seq,
// D/8], params fp32 [B, H_kv, max_seq, 2].  Keys and values are quantised in
// one call.  D a multiple of 8 up to 256.
void write_kv4_inplace(Tensor& k_codes, Tensor& k_params, Tensor& v_codes, Tensor& v_params,
                       const Tensor& k, const Tensor& v, int pos);
Tensor read_kv4_expanded(const Tensor& codes, const Tensor& params, int valid_len, int group);

}  // namespace ctd::ops
