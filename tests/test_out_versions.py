"""What a call writes into a caller's tensor is an in-place change to autograd: a backward pass that still needs what the
tensor held raises, as behind torch's own ``out=``, instead of reading the new rows."""

import pytest
import torch

from sgl_asap_amd.moe import linear as L
from sgl_asap_amd.moe import sort as S
from sgl_asap_amd.moe.linear import Int8Linear
from sgl_asap_amd.moe.sort import sort_tokens, unsort_tokens

CHANGED = "inplace operation"


@pytest.fixture
def on_host(monkeypatch):
    """The Python of the calls on the CPU, with launches that do nothing."""
    for module in (L, S):
        monkeypatch.setattr(module, "need_gpu", lambda *a: None)
        monkeypatch.setattr(module, "launch", lambda *a: None)


def check_saved(buf, write):
    """write() changes buf (or rows of it), which a product saved before."""
    w = torch.ones(buf.shape[1], device=buf.device, dtype=buf.dtype, requires_grad=True)
    y = buf @ w
    before = buf._version
    write()
    assert buf._version > before
    with pytest.raises(RuntimeError, match=CHANGED):
        y.sum().backward()


def test_sorted_rows_into_a_buffer(on_host):
    ids = torch.zeros(4, 2, dtype=torch.int32)
    buf = torch.zeros(9, 16)
    check_saved(buf, lambda: sort_tokens(torch.zeros(4, 16), ids, 3, out=buf))
    check_saved(buf, lambda: sort_tokens(torch.zeros(4, 16), ids, 3, out=buf[1:]))


def test_dense_products_into_a_buffer(on_host):
    layer = Int8Linear(torch.zeros(24, 16, dtype=torch.int8), torch.zeros(24))
    fp8 = L.Fp8BlockLinear(torch.zeros(24, 16, dtype=torch.uint8), torch.zeros(1, 1))
    for f in (layer, fp8):
        buf = torch.zeros(5, 24, dtype=torch.bfloat16)
        check_saved(buf, lambda: f(torch.zeros(5, 16, dtype=torch.bfloat16), out=buf))
        check_saved(buf, lambda: f.silu_mul(torch.zeros(5, 32, dtype=torch.bfloat16), out=buf))
        check_saved(buf, lambda: f(torch.zeros(3, 16, dtype=torch.bfloat16), out=buf[1:4]))


def test_buffers_of_inference_mode(on_host):
    """They have no version, and no backward pass may hold them."""
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with torch.inference_mode():
        buf = torch.zeros(8, 16)
        assert sort_tokens(torch.zeros(4, 16), ids, 3, out=buf)[0] is buf
    with torch.no_grad():
        assert sort_tokens(torch.zeros(4, 16), ids, 3, out=buf)[0] is buf


@pytest.mark.gpu
def test_a_buffer_that_a_second_batch_took():
    """unsort_tokens with trainable weights saves the rows; the next batch sorted into them is not what its backward reads."""
    from gpu_util import dev, say

    say("a buffer's second batch")
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20, 32, generator=g).to(dev())
    ids = torch.randint(0, 4, (20, 2), generator=g).int().to(dev())
    w = torch.rand(20, 2, generator=g).to(dev()).requires_grad_()
    buf = torch.zeros(40, 32, device=dev())
    rows, order = sort_tokens(x, ids, 4, out=buf)
    y = unsort_tokens(rows, order, w)
    (want,) = torch.autograd.grad(y.sum(), w, retain_graph=True)
    assert torch.equal(want, torch.autograd.grad(unsort_tokens(rows.clone(), order, w).sum(), w)[0])
    sort_tokens(-x, ids, 4, out=buf)
    with pytest.raises(RuntimeError, match=CHANGED):
        y.sum().backward()
