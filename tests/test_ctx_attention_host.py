"""CPU tests of the attention operators' refusals: the C entry points check
their arguments before they touch a device, and the Python calls check their
tensors before the C call."""

import ctypes

import pytest

torch = pytest.importorskip("torch")


class Rows(ctypes.Structure):  # irt_rows
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class AttnArgs(ctypes.Structure):  # irt_attn_args
    _fields_ = [
        ("device", ctypes.c_int32), ("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("num_seqs", ctypes.c_int32), ("max_q_len", ctypes.c_int32),
        ("max_k_len", ctypes.c_int32), ("scale", ctypes.c_float), ("q_rows", ctypes.c_int64),
        ("seqs", ctypes.c_void_p), ("q", Rows), ("gate", Rows), ("out", Rows), ("key_mask", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
    ]


class Cache(ctypes.Structure):  # irt_kv4_cache
    _fields_ = [("rows", ctypes.c_int64), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p)]


@pytest.fixture()
def ops(pkg):
    if not pkg.LIB_PATH.exists():
        pytest.skip("library not built")
    pkg.lib()
    import irodori_b200.ops as o
    return o


def attn_args(o, **kw):
    """A valid call's arguments over made-up addresses (never read: each test breaks one of them)."""
    a = AttnArgs(device=0, dtype=0, heads=4, kv_heads=2, head_dim=128, num_seqs=2, max_q_len=3, max_k_len=5,
                    scale=0.1, q_rows=6, seqs=None, q=Rows(0x10000000, 512, 128), gate=Rows(),
                    out=Rows(0x20000000, 512, 128), key_mask=None, lse=None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def status(pkg, rc):
    return pkg.STATUS_NAMES.get(rc, rc), pkg.lib().irt_last_error().decode()


K, V = (0x30000000, 256, 128), (0x40000000, 256, 128)

BAD = [
    (dict(dtype=2), "InvalidArgument", "dtype"),
    (dict(heads=3), "Shape", "multiple of kv_heads"),
    (dict(heads=0), "Shape", "multiple of kv_heads"),
    (dict(kv_heads=0), "Shape", "multiple of kv_heads"),
    (dict(head_dim=100), "Shape", "head_dim 100"),
    (dict(head_dim=264), "Shape", "head_dim 264"),
    (dict(head_dim=0), "Shape", "head_dim 0"),
    (dict(num_seqs=-1), "Shape", "num_seqs"),
    (dict(num_seqs=65536), "Shape", "num_seqs"),
    (dict(max_q_len=-1), "Shape", "must not be negative"),
    (dict(max_k_len=-1), "Shape", "must not be negative"),
    (dict(max_q_len=4), "Shape", "without a sequence table"),
    (dict(max_k_len=6), "Shape", "without a sequence table"),
    (dict(q_rows=1 << 30), "Shape", "2^30"),
    (dict(q_rows=-1), "Shape", "2^30"),
    (dict(scale=float("nan")), "InvalidArgument", "scale"),
    (dict(scale=float("inf")), "InvalidArgument", "scale"),
    (dict(q=(0, 512, 128)), "InvalidArgument", "q is NULL"),
    (dict(out=(0, 512, 128)), "InvalidArgument", "out is NULL"),
    (dict(q=(0x10000001, 512, 128)), "InvalidArgument", "q is not aligned"),
    (dict(q=(0x10000000, -512, 128)), "Shape", "negative stride"),
    (dict(q=(0x10000000, 1 << 50, 128)), "Shape", "2^48"),
    (dict(out=(0x20000000, 128, 128)), "Shape", "overlap one another"),
    (dict(out=(0x20000000, 512, 64)), "Shape", "overlap one another"),
    (dict(out=(0x10000000, 512, 128)), "InvalidArgument", "out overlaps q"),
    (dict(out=(0x30000000 + 100, 512, 128)), "InvalidArgument", "out overlaps k"),
    (dict(gate=(0x20000000 + 64, 512, 128)), "InvalidArgument", "out overlaps gate"),
]


@pytest.mark.parametrize("kw,kind,msg", BAD)
def test_cross_attention_refusals_through_the_c_abi(pkg, ops, kw, kind, msg):
    a = attn_args(ops, **{k: Rows(*v) if isinstance(v, tuple) else v for k, v in kw.items()})
    k, v = Rows(*K), Rows(*V)
    rc = pkg.lib().irt_cross_attention(ctypes.byref(a), ctypes.byref(k), ctypes.byref(v), 10, None)
    got, text = status(pkg, rc)
    assert got == kind and msg in text, (got, text)


def cache_struct(ops, **kw):
    c = Cache(10, 2, 128, 0x50000000, 0x51000000, 0x52000000, 0x53000000)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,kind,msg", [
    (dict(kv_heads=4), "Shape", "the cache holds 4 heads"),
    (dict(head_dim=64), "Shape", "heads of 64"),
    (dict(rows=-1), "Shape", "context rows"),
    (dict(k_scales=None), "InvalidArgument", "cache buffer is NULL"),
    (dict(v_codes=0x52000008), "InvalidArgument", "aligned to 16"),
])
def test_kv4_attention_refusals_through_the_c_abi(pkg, ops, kw, kind, msg):
    a, c = attn_args(ops), cache_struct(ops, **kw)
    rc = pkg.lib().irt_kv4_attention(ctypes.byref(a), ctypes.byref(c), None, None, None)
    got, text = status(pkg, rc)
    assert got == kind and msg in text, (got, text)


def test_kv4_attention_needs_both_own_tensors(pkg, ops):
    a, c, r = attn_args(ops), cache_struct(ops), Rows(*K)
    rc = pkg.lib().irt_kv4_attention(ctypes.byref(a), ctypes.byref(c), ctypes.byref(r), None, None)
    got, text = status(pkg, rc)
    assert got == "MissingInput" and "go together" in text


@pytest.mark.parametrize("start,n,src,kind,msg", [
    (-1, 3, 5, "Shape", "outside the cache"), (8, 3, 5, "Shape", "outside the cache"),
    (0, -1, 5, "Shape", "outside the cache"), (11, 0, 5, "Shape", "outside the cache"),
    (2 ** 62, 2 ** 62, 5, "Shape", "outside the cache"), (0, 6, 5, "Shape", "exceeds the source"),
    (0, 3, -1, "Shape", "source rows"),
])
def test_kv4_append_refusals_through_the_c_abi(pkg, ops, start, n, src, kind, msg):
    c, k, v = cache_struct(ops), Rows(*K), Rows(*V)
    rc = pkg.lib().irt_kv4_append(0, 0, ctypes.byref(c), start, n, ctypes.byref(k), ctypes.byref(v), src, None, None)
    got, text = status(pkg, rc)
    assert got == kind and msg in text, (got, text)


def test_kv4_read_refuses_outputs_that_overlap(pkg, ops):
    c, k, v = cache_struct(ops), Rows(0x30000000, 128, 128), Rows(*V)
    rc = pkg.lib().irt_kv4_read(0, 0, ctypes.byref(c), 0, 5, ctypes.byref(k), ctypes.byref(v), None)
    got, text = status(pkg, rc)
    assert got == "Shape" and "overlap one another" in text


def test_the_python_calls_pack_the_headers_structures(ops):
    assert (ops._ROWS.size, ops._ATTN.size, ops._CACHE.size) == tuple(map(ctypes.sizeof, (Rows, AttnArgs, Cache)))
    a = AttnArgs.from_buffer_copy(ops._ATTN.pack(*range(1, 9), 0.5, *range(10, 23)))
    assert (a.device, a.max_k_len, a.scale, a.q_rows, a.seqs, a.q.data, a.q.head_stride, a.gate.data, a.out.data,
            a.out.row_stride, a.key_mask, a.lse) == (1, 8, 0.5, 10, 11, 12, 14, 15, 18, 19, 21, 22)
    c = Cache.from_buffer_copy(ops._CACHE.pack(*range(1, 8)))
    assert (c.rows, c.kv_heads, c.head_dim, c.k_codes, c.v_scales) == (1, 2, 3, 4, 7)


def test_null_arguments(pkg, ops):
    L, a, r, c = pkg.lib(), attn_args(ops), Rows(*K), cache_struct(ops)
    assert L.irt_cross_attention(None, ctypes.byref(r), ctypes.byref(r), 10, None) == 22
    assert L.irt_cross_attention(ctypes.byref(a), None, ctypes.byref(r), 10, None) == 22
    assert L.irt_kv4_attention(ctypes.byref(a), None, None, None, None) == 22
    assert L.irt_kv4_append(0, 0, None, 0, 1, ctypes.byref(r), ctypes.byref(r), 1, None, None) == 22
    assert L.irt_kv4_read(0, 0, ctypes.byref(c), 0, 1, None, ctypes.byref(r), None) == 22


def test_python_calls_refuse_host_tensors(pkg, ops):
    q = torch.zeros(3, 4, 128)
    for call in (lambda: pkg.cross_attention(q, q, q, None, 3, 3), lambda: pkg.kv4_append(None, q, q),
                 lambda: pkg.Kv4Cache.from_buffers(q, q, q, q)):
        with pytest.raises(pkg.IrodoriError) as ei:
            call()
        assert ei.value.kind == "InvalidArgument" and "CUDA tensor" in str(ei.value)
    for bad in ((-1, 2, 128), (5, 0, 128), (5, 2, 12), (5, 2, 264)):
        with pytest.raises(pkg.IrodoriError) as ei:
            pkg.Kv4Cache(*bad)
        assert ei.value.kind == "Shape"
    for lens in (([1], [1, 2]), ([-1], [2]), ([1], [-2])):
        with pytest.raises(pkg.IrodoriError) as ei:
            pkg.attention_table(*lens)
        assert ei.value.kind == "Shape"
    with pytest.raises(pkg.IrodoriError):
        pkg.attention_table([1], [1], [1, 2])


def test_what_is_written_must_lie_apart(pkg, ops):
    """lse, the mask and the cache's buffers against what a call writes; columns of one tensor are apart."""
    L = pkg.lib()
    byref = ctypes.byref

    def refusal(rc):
        got, text = status(pkg, rc)
        assert got == "InvalidArgument", (got, text)
        return text

    k, v = Rows(*K), Rows(*V)
    for kw, msg in ((dict(lse=0x20000000), "out overlaps lse"), (dict(lse=0x10000000), "lse overlaps q"),
                    (dict(lse=0x30000000), "lse overlaps k"), (dict(key_mask=0x20000004), "out overlaps key_mask"),
                    (dict(seqs=0x20000010), "out overlaps seqs"), (dict(lse=0x60000002), "aligned to 4"),
                    (dict(seqs=0x60000002), "aligned to 4")):
        assert msg in refusal(L.irt_cross_attention(byref(attn_args(ops, **kw)), byref(k), byref(v), 10, None))
    a = attn_args(ops, out=Rows(0x51000000, 512, 128))
    assert "out overlaps k_scales" in refusal(L.irt_kv4_attention(byref(a), byref(cache_struct(ops)), None, None, None))
    # 10 rows x 2 heads x 64 bytes of codes: 1280 bytes
    for kw, msg in ((dict(v_codes=0x50000000 + 1264), "k_codes overlaps the cache's v_codes"),
                    (dict(k_scales=0x50000000), "k_codes overlaps the cache's k_scales"),
                    (dict(v_scales=0x30000000), "k overlaps the cache's v_scales"),
                    (dict(k_codes=0x40000000), "v overlaps the cache's k_codes")):
        c = cache_struct(ops, **kw)
        assert msg in refusal(L.irt_kv4_append(0, 0, byref(c), 0, 5, byref(k), byref(v), 5, None, None))
    c = cache_struct(ops)
    assert "source index overlaps" in refusal(
        L.irt_kv4_append(0, 0, byref(c), 0, 5, byref(k), byref(v), 5, 0x50000000, None))
    assert "k overlaps v" in refusal(L.irt_kv4_read(0, 0, byref(c), 0, 5, byref(k), byref(k), None))
    # columns of one tensor pass the check that a shared column fails (the call then stops at its lse)
    wide = [Rows(0x10000000 + 2 * 256 * i, 768, 128) for i in range(3)]
    for q, out, msg in ((0, 1, "lse overlaps k"), (1, 0, "lse overlaps k"), (2, 0, "lse overlaps k"),
                        (1, 1, "out overlaps q")):
        a = attn_args(ops, heads=2, kv_heads=2, q=wide[q], out=wide[out], lse=0x30000000)
        assert refusal(L.irt_cross_attention(byref(a), byref(k), byref(v), 10, None)) == msg


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38])
def test_a_scale_that_the_kernels_cannot_hold(pkg, ops, scale):
    a, k, v = attn_args(ops, scale=scale), Rows(*K), Rows(*V)
    got, text = status(pkg, pkg.lib().irt_cross_attention(ctypes.byref(a), ctypes.byref(k), ctypes.byref(v), 10, None))
    assert got == "InvalidArgument" and "scale" in text


def test_python_ranges_that_c_integers_would_wrap(pkg, ops):
    c = pkg.Kv4Cache.__new__(pkg.Kv4Cache)
    c.rows = 10
    for start, n in ((2 ** 64, 1), (0, 2 ** 64), (-1, 1), (11, 0), (3, 8), (-(2 ** 64), 2)):
        with pytest.raises(pkg.IrodoriError) as ei:
            ops._row_range(c, start, n)
        assert ei.value.kind == "Shape" and "outside the cache" in str(ei.value)
    ops._row_range(c, 10, 0)
    with pytest.raises(pkg.IrodoriError):
        ops._row_range(None, 0, 0)
    for lens in (([2 ** 29, 2 ** 29], [1, 1]), ([1], [2 ** 31]), ([1, 1], [2 ** 29, 2 ** 29])):
        with pytest.raises(pkg.IrodoriError) as ei:
            pkg.attention_table(*lens)
        assert ei.value.kind == "Shape" and "2^30" in str(ei.value)
    for starts in ([2 ** 31], [-1]):
        with pytest.raises(pkg.IrodoriError) as ei:
            pkg.attention_table([1], [1], starts)
        assert ei.value.kind == "Shape"
