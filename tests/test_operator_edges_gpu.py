"""The named operators at the edges of what they accept, on the GPU, against 64-bit forms (operators_reference.py)."""
import ctypes as C

import pytest
import torch

import operators_reference as ref
import test_operator_kernels_gpu as direct
import test_operators_gpu as program
from ryft_b200 import kernels as K
from ryft_b200 import pjrt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def client():
    c = pjrt.load_cuda_13_plugin().client({"visible_devices": [0]})
    yield c
    c.close()


@pytest.fixture(scope="module")
def lib():
    return K.load()


# ---- no query heads -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("documents", [False, True])
def test_key_heads_without_query_heads_have_gradients_of_zero(lib, documents):
    B, Hk, S, D = 2, 3, 200, 72
    q, k, v, do = direct.make(1, B, 0, Hk, S, S, D)
    o, lse = torch.empty_like(q), torch.empty(B, 0, S, device="cuda")
    grads = (do, torch.empty_like(q), torch.full_like(k, 7.0), torch.full_like(v, 7.0))
    options = {"documents": torch.zeros(B, S, dtype=torch.int32, device="cuda")} if documents else {}
    a = direct.attention_args(lib, q, k, v, o, lse, grads, causal=1, **options)
    before = lib.b2x_kernel_launch_count()
    rc, status = direct.launch(lib, a, True)
    torch.cuda.synchronize()
    assert rc == 0 and not status.item()
    assert lib.b2x_kernel_launch_count() - before == lib.b2x_head_attention_launches(C.byref(a), 1)
    assert not grads[2].any() and not grads[3].any()
