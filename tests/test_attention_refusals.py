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
