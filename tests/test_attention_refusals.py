"""CPU tests of further refusals of the attention operators (the C entry points check their arguments before they touch
a device)."""

import ctypes

import pytest

from test_ctx_attention_host import K, V, Rows, attn_args, cache_struct, ops, status  # noqa: F401  (fixture)

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("index", [0x60000001, 0x60000002, 0x60000003])
def test_a_source_index_that_is_not_aligned(pkg, ops, n, index):  # noqa: F811
    c, k, v = cache_struct(ops), Rows(*K), Rows(*V)
    rc = pkg.lib().irt_kv4_append(0, 0, ctypes.byref(c), 0, n, ctypes.byref(k), ctypes.byref(v), 5, index, None)
    got, text = status(pkg, rc)
    assert got == "InvalidArgument" and "source index must be aligned to 4 bytes" in text, (got, text)


def test_tensors_with_a_gradient_or_a_tangent(pkg, ops):  # noqa: F811
    """The checks that every tensor goes through, on tensors of the host (device -1)."""
    import torch.autograd.forward_ad as forward_ad

    ops._t()
    x, tangent = torch.randn(3, 2, 8), torch.ones(3, 2, 8)
    plain = (x.data_ptr(), 16, 8)
    checks = (lambda t: ops._heads("q", t, -1, torch.float32, (3, 2, 8)),
              lambda t: ops._plain("k_scales", t, -1, (torch.float32,), (3, 2, 8)))

    def refused(call, what):
        with pytest.raises(pkg.IrodoriError) as ei:
            call()
        assert ei.value.kind == "UnsupportedMode" and what in str(ei.value), str(ei.value)

    for check, want in zip(checks, (plain, plain[0])):
        assert check(x) == want
        leaf = x.detach().requires_grad_()
        refused(lambda: check(leaf), "requires a gradient")
        with torch.no_grad():
            assert check(leaf) == want
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, tangent)
            refused(lambda: check(dual), "forward-mode tangent")
            with torch.no_grad():  # turns reverse mode off, not this
                refused(lambda: check(dual), "forward-mode tangent")
            assert check(forward_ad.unpack_dual(dual).primal) == want
            assert check(x) == want


def test_tracing(pkg, ops):  # noqa: F811
    x = torch.randn(3, 2, 8)
    for call in (lambda t: pkg.cross_attention(t, t, t, None, 3, 3), lambda t: pkg.kv4_append(None, t, t),
                 lambda t: pkg.kv4_read(None), lambda t: pkg.kv4_attention(t, None, None, 3, 3)):
        with pytest.raises(pkg.IrodoriError) as ei:
            torch.jit.trace(call, (x,))
        assert ei.value.kind == "UnsupportedMode" and "trace" in str(ei.value)
