"""What bringing a model's weights into 4 bits leaves to others: models that share its tensors, their
gradients, memory."""
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import trainer as TR  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def test_cpp_api_tests():
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_mx4_model_tests")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr


def test_memory_goes_back_to_the_driver():
    """What the allocator holds shrinks with what lives: beside it, segments that a few 4-bit
    buffers lie in, each of the size of an fp32 weight (4 MB at most here, 126 MB in all) or of
    2 MB for the small ones."""
    c = TR.make_config(vocab_size=512, hidden_size=512, intermediate_size=2048, num_layers=8,
                       num_heads=4, num_kv_heads=2, head_dim=128, rms_norm_eps=1e-5, rope_theta=1e4)
    TR.empty_cache()
    base = TR.memory().reserved
    tr = TR.Trainer(c, seed=0)
    before = TR.memory().reserved - base
    assert before >= 125 * 10 ** 6
    for table in (False, True):
        live = TR.memory().allocated
        tr.quantize_weights(table)
        m = TR.memory()
        assert m.allocated < live
        assert m.reserved - base <= m.allocated + (2 * 4 + 4 * 2 << 20)
    tr.close()


@pytest.mark.parametrize("steps,room", [(0, 0), (0, 16 << 20), (1, 0)])
def test_a_failure_changes_nothing(steps, room):
    """No memory for the first 4-bit weight, or for one further on (40 MB are needed)."""
    c = TR.make_config(vocab_size=512, hidden_size=2048, intermediate_size=4096, num_layers=2,
                       num_heads=16, num_kv_heads=8, head_dim=128, rms_norm_eps=1e-5, rope_theta=1e4)
    ids = np.random.default_rng(1).integers(0, 512, (1, 9))
    losses = []
    for fails in (False, True):
        tr = TR.Trainer(c, seed=0)
        tr.set_batch(ids, ids)
        if steps:
            tr.make_optimizer()
            tr.train_step()
        if fails:
            TR.empty_cache()
            TR.set_memory_limit(TR.memory().reserved + room)
            try:
                with pytest.raises(TR.CtdError):
                    tr.quantize_weights(True)
            finally:
                TR.set_memory_limit(0)
        if not steps:
            tr.make_optimizer()
        run = [tr.train_step().loss, tr.forward_backward(False)]
        tr.quantize_weights(True)
        losses.append(run + [tr.forward_backward(False)])
        tr.close()
    assert losses[0] == losses[1]
