"""GPU tests of the attention operators over context states (cross attention,
attention over the 4-bit cache) and of the cache itself, against their
definitions in 64 bits."""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = {BF: 2.0 ** -8, F32: 2.0 ** -24}  # largest relative error of one rounding


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch.device("cuda:0")


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def reference(q, ctx_k, ctx_v, seqs, scale, mask=None, gate=None, ks=None, vs=None):
    """(out, lse, tolerance of out, tolerance of lse, covered rows) in 64 bits.

    With u the error of one rounding to the output type, A = sum_j p_j |v_j|
    (p normalised) and e = 2^-24: a score is a sum of hd products in f32, off
    by at most d = (hd + 2) e sum|q k| scale and by e times a few for the
    scaling, so each p_j moves by a factor exp(d) in the numerator and in the
    sum; the exponential itself is within 2^-21; sums of n terms add n e each.
    p_j is rounded to bf16 before the second product where the operands are
    bf16 (u again); the result is rounded once.
      |out error| <= u |out| + A (u_p + 2 d + 2 (n + 8) e + 2^-20)
      |lse error| <= d + (n + 8) e + 2^-20 + 4 e |lse|
    (first order; a factor 1.01 covers the products of small terms.)
    """
    n, h, hd = q.shape
    hkv = ctx_k.shape[1] if ctx_k is not None else ks.shape[1]
    u, e = U[q.dtype], 2.0 ** -24
    up = u if q.dtype == BF else 0.0
    out = torch.zeros(n, h, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((n, h), -math.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros(n, h, dtype=torch.float64, device=q.device)
    covered = torch.zeros(n, dtype=torch.bool, device=q.device)
    for q0, ql, k0, kl in seqs:
        covered[q0:q0 + ql] = True
        k, v = ctx_k[k0:k0 + kl].double(), ctx_v[k0:k0 + kl].double()
        if mask is not None:
            keep = mask[k0:k0 + kl].bool()
            k, v = k[keep], v[keep]
        if ks is not None:
            k, v = torch.cat([ks[q0:q0 + ql].double(), k]), torch.cat([vs[q0:q0 + ql].double(), v])
        nk = k.shape[0]
        if nk == 0 or ql == 0:
            continue
        k, v = (x.repeat_interleave(h // hkv, 1).transpose(0, 1) for x in (k, v))  # [h, nk, hd]
        qq = q[q0:q0 + ql].double().transpose(0, 1)
        s = qq @ k.transpose(1, 2) * scale
        d = (hd + 8) * e * ((qq.abs() @ k.abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        o, a = p @ v, p @ v.abs()
        ls = torch.logsumexp(s, -1)
        t = u * o.abs() + a * (up + 2 * d + 2 * (nk + 8) * e + 2.0 ** -20)
        out[q0:q0 + ql], tol[q0:q0 + ql] = o.transpose(0, 1), 1.01 * t.transpose(0, 1)
        lse[q0:q0 + ql] = ls.T
        ltol[q0:q0 + ql] = 1.01 * (d.squeeze(-1) + (nk + 8) * e + 2.0 ** -20 + 4 * e * ls.abs()).T
    if gate is not None:
        g = gate.double()
        out, tol = out * g, tol * g.abs() * (1 + 2 * e)
    # the smallest normal number of the output type: what underflow may lose
    return out, lse, tol + 1.2e-38, ltol, covered


def check(got, lse, ref, fill=None):
    out, rl, tol, ltol, cov = ref
    err = (got.double() - out).abs()
    bad = ~(err <= tol) & cov[:, None, None]
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float((err / tol)[cov].max()):.3f} of the tolerance"
    if fill is not None:
        assert (got[~cov] == fill).all()
    if lse is not None:
        none = torch.isinf(rl) & cov[:, None]
        assert (lse[none] == -math.inf).all()
        ok = ~torch.isinf(rl) & cov[:, None]
        le = (lse.double() - rl).abs()[ok]
        assert (le <= ltol[ok]).all(), float((le / ltol[ok]).max())


def table(q_lens, k_lens, q_gap=0, k_gap=0):
    rows, q, k = [], 0, 0
    for a, b in zip(q_lens, k_lens):
        rows.append((q, a, k, b))
        q, k = q + a + q_gap, k + b + k_gap
    return rows, q, k


def device_table(seqs, dev):
    return torch.tensor(seqs, dtype=torch.int32, device=dev).reshape(-1, 4)


def make_cache(pkg, rows, hkv, hd, g, dev, dtype=F32):
    """(cache, the K and V values that it holds)."""
    c = pkg.Kv4Cache(rows, hkv, hd)
    k = torch.randn(rows, hkv, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(rows, hkv, hd, device=dev, generator=g).to(dtype)
    pkg.kv4_append(c, k, v)
    return (c, *pkg.kv4_read(c, dtype=F32))


# (head_dim, heads, kv_heads)
HEADS = [(128, 16, 16), (128, 4, 1), (64, 6, 2), (128, 8, 1), (8, 4, 4), (96, 3, 3), (40, 10, 2), (256, 2, 1), (136, 2, 2),
         (128, 32, 2)]
# (query lengths, context lengths)
LENGTHS = [([1], [1]), ([1], [577]), ([1, 1, 1], [300, 0, 1]), ([3, 1, 7, 2], [65, 64, 63, 129]),
           ([130, 1, 0, 64], [70, 200, 5, 0]), ([200, 33], [700, 129]), ([5], [3001])]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd,h,hkv", HEADS)
@pytest.mark.parametrize("q_lens,k_lens", LENGTHS)
def test_cross_attention(pkg, dev, dtype, hd, h, hkv, q_lens, k_lens):
    seqs, nq, nk = table(q_lens, k_lens)
    g = gen(dev, 1000 * hd + 7 * h + sum(q_lens) + sum(k_lens))
    q = torch.randn(nq, h, hd, device=dev, generator=g).to(dtype)
    k = torch.randn(nk, hkv, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(nk, hkv, hd, device=dev, generator=g).to(dtype)
    out, lse = pkg.cross_attention(q, k, v, device_table(seqs, dev), max(q_lens), max(k_lens), return_lse=True)
    pkg.attention_check(0)
    check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd,h,hkv", HEADS)
@pytest.mark.parametrize("q_lens,k_lens", LENGTHS)
@pytest.mark.parametrize("own_rows", [False, True])
def test_kv4_attention(pkg, dev, dtype, hd, h, hkv, q_lens, k_lens, own_rows):
    seqs, nq, nk = table(q_lens, k_lens)
    g = gen(dev, 1000 * hd + 7 * h + sum(q_lens) + sum(k_lens) + own_rows)
    q = torch.randn(nq, h, hd, device=dev, generator=g).to(dtype)
    cache, ck, cv = make_cache(pkg, nk, hkv, hd, g, dev)
    ks = vs = None
    if own_rows:
        ks = torch.randn(nq, hkv, hd, device=dev, generator=g).to(dtype)
        vs = torch.randn(nq, hkv, hd, device=dev, generator=g).to(dtype)
    out, lse = pkg.kv4_attention(q, cache, device_table(seqs, dev), max(q_lens), max(k_lens), k_self=ks, v_self=vs,
                                 return_lse=True)
    pkg.attention_check(0)
    check(out, lse, reference(q, ck, cv, seqs, 1 / math.sqrt(hd), ks=ks, vs=vs))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("q_lens,h,hkv", [([1, 1, 2], 16, 16), ([150, 20, 1], 4, 2)])
def test_mask_gate_and_whatever_lies_outside(pkg, dev, dtype, four_bit, q_lens, h, hkv):
    """Masked rows, rows between and behind the sequences and outputs that no
    sequence covers hold NaN and infinities: none of it is read or touched.
    The last sequence's mask leaves nothing."""
    hd = 128
    k_lens = [130, 577, 90]
    seqs, nq, nk = table(q_lens, k_lens, q_gap=3, k_gap=5)
    g = gen(dev, 11 + len(q_lens) + h + four_bit)
    q = torch.full((nq, h, hd), float("nan"), device=dev, dtype=dtype)
    gate = torch.full((nq, h, hd), float("nan"), device=dev, dtype=dtype)
    k = torch.full((nk, hkv, hd), float("nan"), device=dev, dtype=dtype)
    v = torch.full((nk, hkv, hd), float("inf"), device=dev, dtype=dtype)
    mask = torch.zeros(nk, dtype=torch.uint8, device=dev)
    for i, (q0, ql, k0, kl) in enumerate(seqs):
        q[q0:q0 + ql] = torch.randn(ql, h, hd, device=dev, generator=g).to(dtype)
        gate[q0:q0 + ql] = torch.rand(ql, h, hd, device=dev, generator=g).to(dtype)
        if i < 2:
            keep = (torch.rand(kl, device=dev, generator=g) < 0.6).nonzero().squeeze(1) + k0
            mask[keep] = 3  # any non-zero value attends
            k[keep] = torch.randn(len(keep), hkv, hd, device=dev, generator=g).to(dtype)
            v[keep] = torch.randn(len(keep), hkv, hd, device=dev, generator=g).to(dtype)
    out = torch.full((nq, h, hd), 7.0, device=dev, dtype=dtype)
    tab = device_table(seqs, dev)
    if four_bit:
        cache = pkg.Kv4Cache(nk, hkv, hd)
        pkg.kv4_append(cache, k, v)
        k, v = pkg.kv4_read(cache, dtype=F32)
        bad = mask == 0
        assert k[bad].isnan().all() and v[bad].isnan().all()
        _, lse = pkg.kv4_attention(q, cache, tab, max(q_lens), max(k_lens), key_mask=mask, gate=gate, out=out,
                                   return_lse=True)
    else:
        _, lse = pkg.cross_attention(q, k, v, tab, max(q_lens), max(k_lens), key_mask=mask, gate=gate, out=out,
                                     return_lse=True)
    pkg.attention_check(0)
    check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd), mask=mask, gate=gate), fill=7.0)
    q0, ql = seqs[2][:2]
    assert (out[q0:q0 + ql] == 0).all()
    # the same mask as bool
    again = torch.full((nq, h, hd), 7.0, device=dev, dtype=dtype)
    if not four_bit:
        pkg.cross_attention(q, k, v, tab, max(q_lens), max(k_lens), key_mask=mask != 0, gate=gate, out=again)
        assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_in_an_attended_row_reaches_its_queries(pkg, dev, dtype):
    g = gen(dev, 5)
    q = torch.randn(140, 2, 128, device=dev, generator=g).to(dtype)
    k = torch.randn(200, 2, 128, device=dev, generator=g).to(dtype)
    v = torch.randn(200, 2, 128, device=dev, generator=g).to(dtype)
    k[150, 1, 3] = float("nan")
    for ql in (2, 140):
        out = pkg.cross_attention(q[:ql], k, v, device_table([(0, ql, 0, 200)], dev), ql, 200)
        assert out[:, 1].isnan().all() and not out[:, 0].isnan().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ql", [2, 70])
def test_strides_and_alignment(pkg, dev, dtype, ql):
    """Head-major tensors, slices of a wider projection and bases that are not
    aligned for vector loads give what their contiguous copies give (to the
    tolerance: another kernel may run)."""
    h, hd, kl = 4, 128, 150
    g = gen(dev, ql)
    seqs = [(0, ql, 0, kl), (ql, ql, 20, kl - 20)]
    tab = device_table(seqs, dev)

    def head_major(n):
        return torch.randn(h, n, hd, device=dev, generator=g).to(dtype).transpose(0, 1)

    def sliced(n):
        return torch.randn(n, 3, h, hd, device=dev, generator=g).to(dtype)[:, 1]

    def odd(n):
        return torch.randn(n * h * hd + 1, device=dev, generator=g).to(dtype)[1:].reshape(n, h, hd)

    def padded(n):  # strides that are no multiple of 16 bytes
        return torch.randn(n, h, hd + 1, device=dev, generator=g).to(dtype)[..., :hd]

    for make in (head_major, sliced, odd, padded):
        q, k, v, gate = make(2 * ql), make(kl), make(kl), make(2 * ql)
        out = make(2 * ql)
        res, lse = pkg.cross_attention(q, k, v, tab, ql, kl, gate=gate, out=out, return_lse=True)
        assert res is out
        check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd), gate=gate))
        cache = pkg.Kv4Cache(kl, h, hd)
        pkg.kv4_append(cache, k, v)
        ck, cv = pkg.kv4_read(cache, dtype=F32)
        ks, vs = make(2 * ql), make(2 * ql)
        out = make(2 * ql)
        _, lse = pkg.kv4_attention(q, cache, tab, ql, kl, k_self=ks, v_self=vs, out=out, return_lse=True)
        check(out, lse, reference(q, ck, cv, seqs, 1 / math.sqrt(hd), ks=ks, vs=vs))
    # one K row for all heads, as an expanded view
    k1 = torch.randn(kl, 1, hd, device=dev, generator=g).to(dtype).expand(kl, h, hd)
    q, v = sliced(2 * ql), sliced(kl)
    out, lse = pkg.cross_attention(q, k1, v, tab, ql, kl, return_lse=True)
    check(out, lse, reference(q, k1, v, seqs, 1 / math.sqrt(hd)))
    pkg.attention_check(0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ql", [1, 40])
def test_bad_table_entries_are_skipped(pkg, dev, dtype, ql):
    g = gen(dev, 3)
    h, hd, nq, nk = 2, 128, 5 * ql, 100
    q = torch.randn(nq, h, hd, device=dev, generator=g).to(dtype)
    k = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
    good = [(0, ql, 10, 60)]
    bad = [(-1, ql, 0, 10), (nq - ql + 1, ql, 0, 10), (ql, ql, 50, 51), (ql, ql, -3, 10), (ql, ql + 1, 0, 10),
           (ql, ql, 0, 81), (2 ** 31 - 1, ql, 2 ** 31 - 1, 10), (ql, -1, 0, 10), (ql, ql, 0, -1)]
    out = torch.full((nq, h, hd), 7.0, device=dev, dtype=dtype)
    pkg.cross_attention(q, k, v, device_table(bad + good, dev), ql, 80, out=out)
    check(out, None, reference(q, k, v, good, 1 / math.sqrt(hd)), fill=7.0)
    cache, ck, cv = make_cache(pkg, nk, h, hd, g, dev)
    out.fill_(7.0)
    pkg.kv4_attention(q, cache, device_table(good + bad, dev), ql, 80, out=out)
    check(out, None, reference(q, ck, cv, good, 1 / math.sqrt(hd)), fill=7.0)
    pkg.attention_check(0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("four_bit", [False, True])
def test_without_a_table_and_overlapping_context(pkg, dev, dtype, four_bit):
    """Equal sequences need no table; guidance variants read sub-ranges of the
    same context rows."""
    g = gen(dev, 17)
    h, hd, b, lq, lk = 4, 128, 3, 50, 77
    q = torch.randn(b * lq, h, hd, device=dev, generator=g).to(dtype)
    k = torch.randn(b * lk, h, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(b * lk, h, hd, device=dev, generator=g).to(dtype)
    if four_bit:
        cache = pkg.Kv4Cache(b * lk, h, hd)
        pkg.kv4_append(cache, k, v)
        k, v = pkg.kv4_read(cache, dtype=F32)
        call = lambda *a, **kw: pkg.kv4_attention(q, cache, *a, **kw)  # noqa: E731
    else:
        call = lambda *a, **kw: pkg.cross_attention(q, k, v, *a, **kw)  # noqa: E731
    same = [(i * lq, lq, i * lk, lk) for i in range(b)]
    out = call(None, lq, lk)
    check(out, None, reference(q, k, v, same, 1 / math.sqrt(hd)))
    assert torch.equal(out, call(device_table(same, dev), lq, lk))
    over = [(0, lq, 0, 2 * lk), (lq, lq, 30, 100), (2 * lq, lq, 30, 0)]
    out, lse = call(device_table(over, dev), lq, 2 * lk, scale=0.3, return_lse=True)
    check(out, lse, reference(q, k, v, over, 0.3))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_scores_and_single_keys(pkg, dev, dtype):
    """Scores of a few hundred: one key takes all the weight, its value comes
    back as it is; and a score range that underflows."""
    g = gen(dev, 23)
    h, hd, nk = 2, 128, 300
    q = (8 * torch.randn(130, h, hd, device=dev, generator=g)).to(dtype)
    k = (8 * torch.randn(nk, h, hd, device=dev, generator=g)).to(dtype)
    v = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
    for ql in (3, 130):
        seqs = [(0, ql, 0, nk)]
        out, lse = pkg.cross_attention(q, k, v, device_table(seqs, dev), ql, nk, return_lse=True)
        check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd)))
        seqs = [(0, ql, 17, 1)]
        out = pkg.cross_attention(q, k, v, device_table(seqs, dev), ql, 1)
        assert torch.equal(out[:ql], v[17].expand(ql, h, hd))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_offsets_beyond_32_bits(pkg, dev, dtype, four_bit):
    """The attended rows lie more than 2^31 elements into the tensor."""
    h, hd = 16, 128
    rows = 2 ** 31 // (h * hd) + 4096 if not four_bit else 2 ** 31 // (hd // 2) // 2 + 4096
    hh = h if not four_bit else 4  # codes: 4 heads x rows x 64 bytes
    g = gen(dev, 29)
    q = torch.randn(33, hh, hd, device=dev, generator=g).to(dtype)
    tail = 400
    k = torch.randn(tail, hh, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(tail, hh, hd, device=dev, generator=g).to(dtype)
    for ql in (1, 33):
        seqs = [(0, ql, rows - tail, tail)]
        if four_bit:
            c = pkg.Kv4Cache(rows, hh, hd)
            pkg.kv4_append(c, k, v, row_start=rows - tail)
            rk, rv = pkg.kv4_read(c, rows - tail, dtype=F32)
            out = pkg.kv4_attention(q, c, device_table(seqs, dev), ql, tail)
            del c
        else:
            kb = torch.empty(rows, hh, hd, device=dev, dtype=dtype)
            vb = torch.empty(rows, hh, hd, device=dev, dtype=dtype)
            kb[rows - tail:], vb[rows - tail:] = k, v
            rk, rv = k, v
            out = pkg.cross_attention(q, kb, vb, device_table(seqs, dev), ql, tail)
            del kb, vb
        check(out, None, reference(q, rk, rv, [(0, ql, 0, tail)], 1 / math.sqrt(hd)))


def quantised(x):
    """The 4-bit cache's definition in 64 bits: what it holds of x [..., hd]."""
    x = x.double()
    out = torch.zeros_like(x)
    for lo in range(0, x.shape[-1], 32):
        t = x[..., lo:lo + 32]
        amax = t.abs().amax(-1, keepdim=True)
        frac, ex = torch.frexp(amax / 7)
        s = torch.ldexp(torch.ceil(frac * 32), ex - 5).clamp(max=1.125 * 2.0 ** 125)
        c = torch.floor(t.abs() / s + 0.5).clamp(max=7) * torch.sign(t)
        val = torch.where(amax < 2.0 ** -100, torch.zeros_like(t), c * s)
        out[..., lo:lo + 32] = torch.where(torch.isfinite(amax), val, torch.full_like(t, float("nan")))
    return out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [8, 40, 64, 128, 256])
def test_kv4_cache_holds_its_definition(pkg, dev, dtype, hd):
    """Bit for bit, over the whole range of exponents and at the borders
    between codes; and the error of a value is at most half a step."""
    g = gen(dev, hd)
    n, h = 517, 3
    x = torch.randn(n, h, hd, device=dev, generator=g)
    x *= torch.exp2(torch.randint(-130, 126, (n, h, 1), device=dev, generator=g).float())
    x[::7] *= torch.randint(0, 2, (x[::7].shape), device=dev, generator=g)
    x[3] = 0
    # borders: multiples of half a scale, with the maximum at 7 scales, and their neighbours
    b = torch.arange(hd, device=dev) % 15 * 0.5
    x[5] = b
    x[6] = -b * 1.0625
    x[7] = torch.nextafter(b, torch.tensor(9.0, device=dev))
    x[8] = torch.nextafter(b, torch.tensor(-9.0, device=dev))
    x[9] = torch.finfo(BF).max
    x[12] = 2.0 ** -100
    x[13] = 2.0 ** -101
    x = x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    x[10, :, 0] = float("nan")
    x[11, :, hd - 1] = -float("inf")
    c = pkg.Kv4Cache(n, h, hd)
    pkg.kv4_append(c, x, x.flip(0))
    want = quantised(x)
    for dt in (F32, BF):
        k, v = pkg.kv4_read(c, dtype=dt)
        assert torch.equal(k.double().nan_to_num(7e99), want.nan_to_num(7e99))
        assert torch.equal(v.double().nan_to_num(7e99), want.flip(0).nan_to_num(7e99))
    assert k[10].isnan().any() and not k[9].isnan().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("exponent", [-99, 0, 124])
def test_every_bf16_value_against_every_maximum(pkg, dev, dtype, exponent):
    """All 128 largest magnitudes of a binade with all bf16 values of the six binades up to it: every border between
    codes that a bf16 value can lie on or next to."""
    sig = torch.arange(128, device=dev, dtype=torch.float64) / 128 + 1
    vals = torch.cat([sig * 2.0 ** (exponent - i) for i in range(6)])
    vals = torch.cat([vals, -vals, torch.zeros(31 - 2 * len(vals) % 31, device=dev, dtype=torch.float64)]).reshape(-1, 31)
    x = torch.empty(128, len(vals), 32, device=dev, dtype=torch.float64)
    x[:, :, 1:] = vals
    top = (sig * 2.0 ** exponent)[:, None, None]
    x = torch.where(x.abs() <= top, x, torch.zeros_like(x))
    x[:, :, 0] = top[:, :, 0]
    x = x.to(dtype)
    assert torch.equal(x.double().abs().amax(-1, keepdim=True), top.expand(-1, len(vals), 1))
    c = pkg.Kv4Cache(128, len(vals), 32)
    pkg.kv4_append(c, x, -x)
    k, v = pkg.kv4_read(c, dtype=F32)
    assert torch.equal(k.double(), quantised(x)) and torch.equal(v.double(), quantised(-x))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_kv4_append_gathers_and_leaves_the_rest(pkg, dev, dtype):
    g = gen(dev, 2)
    h, hd = 5, 96
    src = torch.randn(90, h, hd, device=dev, generator=g).to(dtype)
    c = pkg.Kv4Cache(200, h, hd)
    first = torch.randn(200, h, hd, device=dev, generator=g).to(dtype)
    pkg.kv4_append(c, first, first)
    idx = torch.tensor([4, 4, -1, 89, 90, 0, 2 ** 31 - 1, -2 ** 31, 7], dtype=torch.int32, device=dev)
    pkg.kv4_append(c, src, src.flip(0), row_start=63, src_rows=idx)
    pkg.kv4_append(c, src[:0], src[:0], row_start=200)
    want_k, want_v = quantised(first), quantised(first)
    for i, j in enumerate(idx.tolist()):
        if 0 <= j < 90:
            want_k[63 + i], want_v[63 + i] = quantised(src[j]), quantised(src.flip(0)[j])
    k, v = pkg.kv4_read(c, dtype=F32)
    assert torch.equal(k.double(), want_k) and torch.equal(v.double(), want_v)
    k, _ = pkg.kv4_read(c, 60, 10, dtype=F32)
    assert torch.equal(k.double(), want_k[60:70])


def test_streams_graphs_and_repeats(pkg, dev):
    """A serving step (append, then attention over own and cached rows) on an
    explicit stream, captured into two graphs that run at the same time, and
    repeated: always the same bits."""
    g = gen(dev, 31)
    h, hd, lq, lk = 16, 128, 30, 400
    q = torch.randn(2 * lq, h, hd, device=dev, generator=g).to(BF)
    ks, vs = torch.randn(2, 2 * lq, h, hd, device=dev, generator=g).to(BF).unbind(0)
    k, v = torch.randn(2, 2 * lk, h, hd, device=dev, generator=g).to(BF).unbind(0)
    tab = pkg.attention_table([lq, lq], [lk, lk])
    one = pkg.attention_table([1] * 4, [lk] * 4, [0, lk, 0, lk])

    def step(cache, out, few, stream=None):
        pkg.kv4_append(cache, k, v, stream=stream)
        pkg.kv4_attention(q, cache, tab, lq, lk, k_self=ks, v_self=vs, out=out, stream=stream)
        pkg.kv4_attention(q[:4], cache, one, 1, lk, out=few, stream=stream)

    def fresh():
        return pkg.Kv4Cache(2 * lk, h, hd), torch.zeros_like(q), torch.zeros_like(q[:4])

    base = fresh()
    step(*base)
    torch.cuda.synchronize()
    ck, cv = pkg.kv4_read(base[0], dtype=F32)
    check(base[1], None, reference(q, ck, cv, tab.tolist(), 1 / math.sqrt(hd), ks=ks, vs=vs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = fresh()
    side.wait_stream(torch.cuda.current_stream())
    step(*other, stream=side)
    side.synchronize()
    assert torch.equal(other[1], base[1]) and torch.equal(other[2], base[2])
    graphs = []
    for _ in range(2):
        bufs = fresh()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(*bufs)
        graphs.append((gr, bufs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for _, bufs in graphs:
        assert torch.equal(bufs[1], base[1]) and torch.equal(bufs[2], base[2])
    for _ in range(10):
        again = fresh()
        step(*again)
        assert torch.equal(again[1], base[1]) and torch.equal(again[2], base[2])
    pkg.attention_check(0)


def test_the_step_agrees_with_attention_over_the_values(pkg, dev):
    """Append -> attention over the cache == cross attention over the values
    that the cache holds (bf16 numbers), to the tolerance of both."""
    g = gen(dev, 37)
    h, hkv, hd = 8, 2, 128
    q_lens, k_lens = [40, 3, 1], [301, 64, 5]
    seqs, nq, nk = table(q_lens, k_lens)
    q = torch.randn(nq, h, hd, device=dev, generator=g).to(BF)
    k = torch.randn(nk, hkv, hd, device=dev, generator=g).to(BF)
    v = torch.randn(nk, hkv, hd, device=dev, generator=g).to(BF)
    c = pkg.Kv4Cache(nk, hkv, hd)
    pkg.kv4_append(c, k, v)
    hk, hv = pkg.kv4_read(c)
    tab = device_table(seqs, dev)
    ref = reference(q, hk, hv, seqs, 1 / math.sqrt(hd))
    for out in (pkg.kv4_attention(q, c, tab, 40, 301), pkg.cross_attention(q, hk, hv, tab, 40, 301)):
        check(out, None, ref)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("ql,scale", [(2, -0.1), (2, 0.0), (75, -0.1), (75, 0.0), (75, 3e-3)])
def test_any_finite_scale(pkg, dev, dtype, four_bit, ql, scale):
    """A negative scale turns the order of the scores, zero makes them equal;
    masked keys stay out of both."""
    g = gen(dev, 41)
    h, hd, nk = 4, 128, 131
    q = torch.randn(ql, h, hd, device=dev, generator=g).to(dtype)
    k = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
    v = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
    mask = (torch.arange(nk, device=dev) % 3 != 0).to(torch.uint8)
    seqs = [(0, ql, 0, nk)]
    tab = device_table(seqs, dev)
    if four_bit:
        c = pkg.Kv4Cache(nk, h, hd)
        pkg.kv4_append(c, k, v)
        k, v = pkg.kv4_read(c, dtype=F32)
        out, lse = pkg.kv4_attention(q, c, tab, ql, nk, key_mask=mask, scale=scale, return_lse=True)
    else:
        out, lse = pkg.cross_attention(q, k, v, tab, ql, nk, key_mask=mask, scale=scale, return_lse=True)
    check(out, lse, reference(q, k, v, seqs, scale, mask=mask))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,kl", [(1, 40), (3, 2000), (40, 64), (64, 1100)])
def test_split_and_unsplit_key_ranges(pkg, dev, dtype, n, kl):
    """From one sequence, whose keys are shared by a cluster, to batches that
    fill the GPU; ragged, with sequences far shorter than the longest."""
    g = gen(dev, n * kl)
    h, hd = 4, 128
    for q_hi in (1, 5, 90):
        r = torch.Generator().manual_seed(n + kl + q_hi)
        ql = [int(x) for x in torch.randint(0, q_hi + 1, (n,), generator=r)]
        kls = [int(x) for x in torch.randint(0, kl + 1, (n,), generator=r)]
        ql[0], kls[-1] = q_hi, kl
        seqs, nq, nk = table(ql, kls)
        q = torch.randn(nq, h, hd, device=dev, generator=g).to(dtype)
        k = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
        v = torch.randn(nk, h, hd, device=dev, generator=g).to(dtype)
        tab = device_table(seqs, dev)
        out, lse = pkg.cross_attention(q, k, v, tab, q_hi, kl, return_lse=True)
        check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd)))
        c = pkg.Kv4Cache(nk, h, hd)
        pkg.kv4_append(c, k, v)
        ck, cv = pkg.kv4_read(c, dtype=F32)
        out, lse = pkg.kv4_attention(q, c, tab, q_hi, kl, return_lse=True)
        check(out, lse, reference(q, ck, cv, seqs, 1 / math.sqrt(hd)))
        ks, vs = torch.randn(2, nq, h, hd, device=dev, generator=g).to(dtype).unbind(0)
        out, lse = pkg.kv4_attention(q, c, tab, q_hi, kl, k_self=ks, v_self=vs, return_lse=True)
        check(out, lse, reference(q, ck, cv, seqs, 1 / math.sqrt(hd), ks=ks, vs=vs))
    pkg.attention_check(0)


@pytest.mark.parametrize("ql", [1, 40])
@pytest.mark.parametrize("size", [2.0 ** 124, 2.0 ** 121, 2.0 ** -90])
def test_kv4_values_at_the_ends_of_the_range(pkg, dev, ql, size):
    """The cache's largest and smallest scales: one key's value comes back as
    the cache holds it (a softmax over one key is 1)."""
    g = gen(dev, 43)
    h, hd = 2, 128
    x = torch.randn(4, h, hd, device=dev, generator=g)
    x = (x / x.abs().amax() * size).to(BF)
    c = pkg.Kv4Cache(4, h, hd)
    pkg.kv4_append(c, torch.randn(4, h, hd, device=dev, generator=g).to(BF), x)
    _, v = pkg.kv4_read(c)
    q = torch.randn(ql, h, hd, device=dev, generator=g).to(BF)
    out = pkg.kv4_attention(q, c, device_table([(0, ql, 2, 1)], dev), ql, 1)
    pkg.attention_check(0)
    assert torch.equal(out, v[2].expand(ql, h, hd))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ql", [2, 70])
def test_out_in_a_column_of_the_packed_projections(pkg, dev, dtype, ql):
    """q, gate and out as columns of one tensor: only out's column changes."""
    g = gen(dev, 91)
    h, hd, n = 4, 64, 3 * ql
    wide = torch.randn(n, 3, h, hd, device=dev, generator=g).to(dtype)
    k, v = torch.randn(2, 300, h, hd, device=dev, generator=g).to(dtype).unbind(0)
    seqs, _, _ = table([ql] * 3, [100, 1, 199])
    before = wide.clone()
    _, lse = pkg.cross_attention(wide[:, 0], k, v, device_table(seqs, dev), ql, 199, gate=wide[:, 2], out=wide[:, 1],
                                 return_lse=True)
    check(wide[:, 1], lse, reference(before[:, 0], k, v, seqs, 1 / math.sqrt(hd), gate=before[:, 2]))
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, 2], before[:, 2])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ql", [1, 50])
def test_tensors_without_rows(pkg, dev, dtype, ql):
    h, hd = 4, 64
    q, none = torch.randn(2 * ql, h, hd, device=dev).to(dtype), torch.empty(0, h, hd, device=dev, dtype=dtype)
    empty, tab = pkg.Kv4Cache(0, h, hd), pkg.attention_table([ql, ql], [0, 0])
    pkg.kv4_append(empty, none, none)
    assert pkg.kv4_read(empty)[0].shape == (0, h, hd)
    for seqs, mk in ((tab, 0), (tab, 70), (None, 0)):
        for out, lse in (pkg.cross_attention(q, none, none, seqs, ql, mk, return_lse=True),
                         pkg.kv4_attention(q, empty, seqs, ql, mk, return_lse=True)):
            assert (out == 0).all() and (lse == -math.inf).all()
    ks, vs = torch.randn(2, 2 * ql, h, hd, device=dev).to(dtype).unbind(0)
    out, lse = pkg.kv4_attention(q, empty, tab, ql, 0, k_self=ks, v_self=vs, return_lse=True)
    check(out, lse, reference(q, none, none, tab.tolist(), 1 / math.sqrt(hd), ks=ks, vs=vs))
    k = torch.randn(5, h, hd, device=dev).to(dtype)
    for seqs in (pkg.attention_table([], []), pkg.attention_table([0, 0], [2, 3])):
        out, lse = pkg.cross_attention(none, k, k, seqs, 3, 3, return_lse=True)
        assert out.shape == (0, h, hd) and lse.shape == (0, h)


def test_python_arguments_out_of_range(pkg, dev):
    q = torch.zeros(2, 4, 64, device=dev)
    tab = pkg.attention_table([2], [2])
    for kw in (dict(max_q_len=2 ** 40), dict(max_k_len=-2 ** 40), dict(scale=1e39), dict(scale=math.inf), dict(v=None),
               dict(v=q.cpu().numpy()), dict(gate=[1.0]), dict(out="q")):
        args = dict(q=q, k=q, v=q, seqs=tab, max_q_len=2, max_k_len=2) | kw
        with pytest.raises(pkg.IrodoriError):
            pkg.cross_attention(**args)
    c = pkg.Kv4Cache(4, 4, 64)
    for call in (lambda: pkg.kv4_append(c, q, q, row_start=2 ** 64), lambda: pkg.kv4_append(c, q, q, row_start=3),
                 lambda: pkg.kv4_read(c, row_start=2 ** 64, rows=1), lambda: pkg.kv4_read(c, rows=5),
                 lambda: pkg.kv4_append(c, q, None), lambda: pkg.kv4_attention(q, None, tab, 2, 2)):
        with pytest.raises(pkg.IrodoriError):
            call()
    assert (pkg.kv4_read(c)[0] == 0).all()


FIRST = """
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("irodori_b200", sys.argv[1], submodule_search_locations=[sys.argv[2]])
pkg = importlib.util.module_from_spec(spec); sys.modules["irodori_b200"] = pkg; spec.loader.exec_module(pkg)
kind = sys.argv[3]
dtype = torch.float32 if kind == "f32" else torch.bfloat16
n = 1 if kind == "few" else 40
torch.manual_seed(1)
q, k = torch.randn(n, 4, 128, device="cuda").to(dtype), torch.randn(90, 4, 128, device="cuda").to(dtype)
tab, cache, out = pkg.attention_table([n], [90]), pkg.Kv4Cache(90, 4, 128), torch.zeros_like(q)
def step():
    pkg.kv4_append(cache, k, k)
    pkg.cross_attention(q, k, k, tab, n, 90, out=out)
    got = pkg.kv4_attention(q, cache, tab, n, 90)
    kk, _ = pkg.kv4_read(cache, dtype=dtype)
    return out, got, kk
torch.cuda.synchronize()
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr):
    captured = step()
gr.replay()
torch.cuda.synchronize()
captured = [x.clone() for x in captured]
for a, b in zip(captured, step()):
    assert torch.equal(a, b) and a.abs().sum() > 0
pkg.attention_check(0)
print("same")
"""


@pytest.mark.parametrize("kind", ["few", "bf16", "f32"])
def test_the_first_calls_of_a_process_may_be_captured(pkg, dev, kind):
    import pathlib
    import subprocess
    import sys

    init = pathlib.Path(pkg.__file__)
    r = subprocess.run([sys.executable, "-c", FIRST, str(init), str(init.parent), kind], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("four_bit,own_rows", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("n", [2, 32, 33, 70, 253, 256, 257])
def test_many_ragged_sequences(pkg, dev, four_bit, own_rows, n):
    """Ragged batches whose sequences have none to four query tiles, with gaps between them, in another order than
    their rows, and entries that are skipped at both ends and inside."""
    g = gen(dev, 95 + n)
    h, hkv, hd, mq, mk = 4, 2, 64, 200, 60
    r = torch.Generator().manual_seed(n)
    ql = torch.randint(0, mq + 1, (n,), generator=r) * (torch.rand(n, generator=r) < 0.8)
    kl = torch.randint(0, mk + 1, (n,), generator=r)
    ql[n // 2], kl[n // 2] = mq, mk
    seqs, nq, nk = table(ql.tolist(), kl.tolist(), 3, 1)
    seqs = [seqs[i] for i in torch.randperm(n, generator=r).tolist()]
    bad = [(0, mq + 1, 0, 1), (nq - 5, 6, 0, 1), (-1, 5, 0, 1), (0, 5, nk - 1, 2), (0, 5, 0, mk + 1), (0, -1, 0, 1)]
    given = list(seqs)
    for i in (0, len(given) // 2, len(given)):  # the batch stays within n + 3 entries
        given.insert(i, bad[(n + i) % len(bad)])
    q = torch.randn(nq, h, hd, device=dev, generator=g).to(BF)
    fill, own = torch.full_like(q, 5.0), {}
    if own_rows:
        own["k_self"], own["v_self"] = torch.randn(2, nq, hkv, hd, device=dev, generator=g).to(BF).unbind(0)
    if four_bit:
        cache, k, v = make_cache(pkg, nk, hkv, hd, g, dev)
        out, lse = pkg.kv4_attention(q, cache, device_table(given, dev), mq, mk, out=fill, return_lse=True, **own)
    else:
        k, v = torch.randn(2, nk, hkv, hd, device=dev, generator=g).to(BF).unbind(0)
        out, lse = pkg.cross_attention(q, k, v, device_table(given, dev), mq, mk, out=fill, return_lse=True)
    check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd), ks=own.get("k_self"), vs=own.get("v_self")), 5.0)
    pkg.attention_check(0)
