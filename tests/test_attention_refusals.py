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


# q and out inside one tensor, as (rows, byte offset of out, row stride, head stride, apart)
SHARED = [
    (6, 256, 512, 256, True),          # [rows, heads, 2, 128]: head by head beside one another
    (6, 256 - 2, 512, 256, False),
    (6, 256 + 2, 512, 256, False),
    (6, 768, 512, 256, True),
    (6, 1536, 128, 1536, True),        # [heads, 2, rows, 128]: the rows of one head, then those of the other tensor
    (6, 1536 - 2, 128, 1536, False),
    (6, 1536 + 2, 128, 1536, False),
    (6, 256, 256, 1536, True),         # [heads, rows, 2, 128]
    (6, 256 + 2, 256, 1536, False),
    (1, 256, 7, 256, True),            # one row: its stride says nothing
    (1, 256 + 2, 7, 256, False),
    (6, 0, 256, 128, False),
]


@pytest.mark.parametrize("rows,offset,row,head,apart", SHARED)
def test_outputs_between_the_values_of_an_input(pkg, ops, rows, offset, row, head, apart):  # noqa: F811
    """Values that share no byte are apart, whatever lies between them (the call then stops at its lse)."""
    q, out = Rows(0x10000000, row, head), Rows(0x10000000 + offset, row, head)
    used = [{at + (i * row + j * head) * 2 + b for i in range(rows) for j in range(2) for b in range(256)} for at in (0, offset)]
    assert used[0].isdisjoint(used[1]) == apart
    a = attn_args(ops, heads=2, kv_heads=2, q=q, out=out, lse=0x30000000, q_rows=rows, num_seqs=1, max_q_len=rows)
    k, v = Rows(*K), Rows(*V)
    got, text = status(pkg, pkg.lib().irt_cross_attention(ctypes.byref(a), ctypes.byref(k), ctypes.byref(v), 10, None))
    assert got == "InvalidArgument" and text == ("lse overlaps k" if apart else "out overlaps q"), (got, text)


def test_a_tensor_without_rows_overlaps_nothing(pkg, ops):  # noqa: F811
    c, k, v = cache_struct(ops), Rows(0x50000000 + 64, 256, 128), Rows(*V)  # inside the cache's codes
    rc = pkg.lib().irt_kv4_append(0, 0, ctypes.byref(c), 0, 0, ctypes.byref(k), ctypes.byref(v), 0, None, None)
    assert rc in (0, 20), status(pkg, rc)  # 20: the checks are passed and there is no GPU
    rc = pkg.lib().irt_kv4_append(0, 0, ctypes.byref(c), 0, 1, ctypes.byref(k), ctypes.byref(v), 1, None, None)
    assert "k overlaps the cache's k_codes" in status(pkg, rc)[1]
