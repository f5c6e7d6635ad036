"""GPU tests of the attention operators' `out` next to torch's autograd."""

import pytest

from test_gpu_ctx_attention import BF, F32, dev  # noqa: F401  (fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("four_bit", [False, True])
def test_autograd_sees_that_out_was_written(pkg, dev, dtype, four_bit):  # noqa: F811
    """A graph that has kept `out` must not use what a later call put there: its backward pass is refused, as after any
    in-place operation of torch's."""
    h, hd, nk, ql = 2, 64, 40, 5
    q = torch.randn(ql, h, hd, device=dev).to(dtype)
    k, v = torch.randn(2, nk, h, hd, device=dev).to(dtype).unbind(0)
    tab, cache = pkg.attention_table([ql], [nk]), pkg.Kv4Cache(nk, h, hd)
    pkg.kv4_append(cache, k, v)

    def call(x, out):
        if four_bit:
            return pkg.kv4_attention(x, cache, tab, ql, nk, out=out)
        return pkg.cross_attention(x, k, v, tab, ql, nk, out=out)

    out = torch.zeros_like(q)
    call(q, out)
    first = out.clone()
    w = torch.ones(hd, device=dev, dtype=dtype, requires_grad=True)
    loss = (out * w).sum()  # keeps out for w's gradient
    loss.backward(retain_graph=True)
    assert torch.allclose(w.grad, first.sum((0, 1)), rtol=0.05, atol=0.05)
    call(2 * q, out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # tensors without a version
        made = torch.empty_like(q)
        assert torch.equal(call(q, made), first)
