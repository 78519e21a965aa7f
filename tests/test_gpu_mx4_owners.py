"""What bringing a model's weights into 4 bits leaves to others: models that share its tensors, their
gradients, memory."""
import os
import subprocess

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
