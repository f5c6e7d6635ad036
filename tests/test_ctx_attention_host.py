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
