"""GPU tests of what the attention operators make of unusual values."""

import math

import pytest

from test_gpu_ctx_attention import BF, F32, check, dev, device_table, gen, reference  # noqa: F401  (fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def own_cache(pkg, rows, h, hd, g, dev, lo, hi):  # noqa: F811
    """A cache over the test's own buffers, with codes in lo..hi and scales of 8 significant bits in [1, 2) (their
    last bit set); and the values c s, exact in 64 bits."""
    bufs, vals = [], []
    for _ in "kv":
        c = torch.randint(lo, hi + 1, (h, rows, hd), device=dev, generator=g)
        s = (1 + (2 * torch.randint(0, 64, (h, rows, -(-hd // 32)), device=dev, generator=g) + 1) / 128).to(BF)
        u = (c + 8).to(torch.uint8)
        bufs += [(u[..., 0::2] | (u[..., 1::2] << 4)).contiguous(), s]
        vals.append((c * s.double().repeat_interleave(32, -1)[..., :hd]).transpose(0, 1).contiguous())
    return (pkg.Kv4Cache.from_buffers(*bufs), *vals)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("ql", [1, 3, 40])
def test_any_bf16_scale_in_f32(pkg, dev, ql, hd):  # noqa: F811
    """c s has up to 11 significant bits, exact in f32: every f32 kernel reads the same values."""
    g = gen(dev, 101 + ql + hd)
    h, nk = 2, 150
    cache, k, v = own_cache(pkg, nk, h, hd, g, dev, -7, 7)
    q = torch.randn(ql, h, hd, device=dev, generator=g)
    seqs = [(0, ql, 0, nk)]
    out, lse = pkg.kv4_attention(q, cache, device_table(seqs, dev), ql, nk, return_lse=True)
    check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd)))
    rk, rv = pkg.kv4_read(cache, dtype=F32)
    assert torch.equal(rk.double(), k) and torch.equal(rv.double(), v)
    rk, rv = pkg.kv4_read(cache)
    assert torch.equal(rk, k.to(BF)) and torch.equal(rv, v.to(BF))


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("ql", [1, 3, 40])
def test_any_bf16_scale_in_bf16(pkg, dev, ql, hd):  # noqa: F811
    """Codes -1, 0 and 1: c s is a bf16 number whatever the scale, so no kernel may round it.  Each query has one key
    (out is its V, lse its score); then all queries have all keys at the same score."""
    g = gen(dev, 201 + ql + hd)
    h, nk = 2, 150
    cache, k, v = own_cache(pkg, nk, h, hd, g, dev, -1, 1)
    q = torch.randn(ql, h, hd, device=dev, generator=g).abs().to(BF)
    for j in (0, 77):
        seqs = [(0, ql, j, 1)]
        out, lse = pkg.kv4_attention(q, cache, device_table(seqs, dev), ql, 1, return_lse=True)
        check(out, lse, reference(q, k, v, seqs, 1 / math.sqrt(hd)))
        assert torch.equal(out, v[j].to(BF).expand(ql, h, hd))
    seqs = [(0, ql, 0, nk)]
    out, lse = pkg.kv4_attention(torch.zeros_like(q), cache, device_table(seqs, dev), ql, nk, return_lse=True)
    check(out, lse, reference(torch.zeros_like(q), k, v, seqs, 1 / math.sqrt(hd)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql,n", [(1, 1), (1, 64), (3, 64), (64, 1), (64, 32)])
def test_large_values_behind_a_maximum_that_rises_late(pkg, dev, dtype, four_bit, hd, ql, n):  # noqa: F811
    """Ten keys have values up to 2^124, all others 0: any sum of weights of at most 1 times values stays below 10 x
    2^124 < 2^128, whatever part of the keys it is over.  Eight of the ten, one in each of the first tiles, weigh 2^-7
    of the two later ones: a kernel whose weights are relative to an earlier maximum would have 2^7 x 2^124."""
    g = gen(dev, 301 + ql + n + hd)
    h, nk = 16, 1024
    top = torch.full((nk,), -40.0, dtype=torch.float64)
    top[5:256:32] = 0.0
    top[131] = top[259] = 7.0
    k = torch.zeros(nk, h, hd, device=dev, dtype=dtype)
    k[:, :, 0] = (top * math.log(2)).to(dev)[:, None].to(dtype)
    v = (torch.rand(nk, h, hd, device=dev, generator=g) * 2 - 1) * 2.0 ** 124
    v[(top < 0).to(dev)] = 0
    v = v.to(dtype)
    q = torch.zeros(n * ql, h, hd, device=dev, dtype=dtype)
    q[:, :, 0] = 1
    seqs = [(i * ql, ql, 0, nk) for i in range(n)]
    tab = device_table(seqs, dev)
    if four_bit:
        cache = pkg.Kv4Cache(nk, h, hd)
        pkg.kv4_append(cache, k, v)
        k, v = pkg.kv4_read(cache, dtype=F32)
        out, lse = pkg.kv4_attention(q, cache, tab, ql, nk, scale=1.0, return_lse=True)
    else:
        out, lse = pkg.cross_attention(q, k, v, tab, ql, nk, scale=1.0, return_lse=True)
    pkg.attention_check(0)
    assert out.isfinite().all()
    check(out, lse, reference(q, k, v, seqs, 1.0))
