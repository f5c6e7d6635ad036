"""Workloads of the attention operators over context states: cross attention to an encoder's states, and the context
cache held in 4 bits (appending to it, reading it back, attention over it).

``run`` computes each of them in its plain form (elementary torch operations in 32 bits, rounded once), or through the
framework's public entry points where ``own`` is true.  Head counts and head dimensions are the framework's default
model (16 heads of 128), its encoders and small test models; sequence lengths are those of a 2 to 30 s utterance
(25 latent frames a second) with 16 to 256 text tokens and a 5 to 15 s speaker reference, and longer contexts.
"""

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

GROUP = 32  # values that share a scale in the 4-bit cache
S_MAX = 2.0 ** 125 * 1.125  # largest scale: 7 * S_MAX is still a bf16 number
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _pkg():
    """The framework's package (its directory's name is not a Python identifier)."""
    if "irodori_b200" not in sys.modules:
        d = Path(__file__).resolve().parents[1] / "irodori-tts-burn_b200"
        spec = importlib.util.spec_from_file_location("irodori_b200", d / "__init__.py",
                                                      submodule_search_locations=[str(d)])
        sys.modules["irodori_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["irodori_b200"])
    return sys.modules["irodori_b200"]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _attn(name, op, nseq, q_lo, q_hi, k_lo, k_hi, heads=16, kv_heads=16, head_dim=128, dtype="bf16", self_keys=False,
          mask=False, gate=False, lse=False):
    c = {"op": op, "nseq": nseq, "q_lo": q_lo, "q_hi": q_hi, "k_lo": k_lo, "k_hi": k_hi, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "self_keys": self_keys, "mask": mask,
         "gate": gate, "lse": lse}
    return {"name": name, **c} if name else c


def _append(name, rows, src_rows, gather, kv_heads=16, head_dim=128, dtype="bf16"):
    c = {"op": "kv4_append", "rows": rows, "src_rows": src_rows, "gather": gather, "kv_heads": kv_heads,
         "head_dim": head_dim, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one frame of one utterance against its text (200) and speaker (376) states: latency
        _attn("cross one frame", "cross", 1, 1, 1, 576, 576),
        # a 30 s utterance, conditional and unconditional copy, gated like the model's attention
        _attn("cross 30 s pair", "cross", 2, 750, 750, 576, 576, gate=True),
        # 64 utterances of 2 to 30 s packed without padding: throughput
        _attn("cross 64 utterances", "cross", 64, 50, 750, 141, 632, gate=True),
        # the last frame of 16 streams against long states: bound by reading them
        _attn("cross 16 streams long", "cross", 16, 1, 1, 5000, 8192, lse=True),
        # grouped heads of 64, padded states under a mask, odd lengths
        _attn("cross grouped masked", "cross", 8, 333, 333, 517, 517, heads=16, kv_heads=4, head_dim=64, mask=True,
              lse=True),
        # the 30 s pair in the fp32 mode
        _attn("cross 30 s pair f32", "cross", 2, 750, 750, 576, 576, dtype="f32", gate=True),
        # one utterance's context rows of one layer, compacted from a padded source on the way in
        _append("append one utterance", 576, 632, True),
        # the context rows of 64 utterances, one layer
        _append("append 64 utterances", 25600, 25600, False),
        # one frame of one utterance against its 4-bit context
        _attn("kv4 one frame", "kv4", 1, 1, 1, 576, 576),
        # 64 utterances, own frames and the 4-bit context: the sampler's attention
        _attn("kv4 64 utterances", "kv4", 64, 50, 750, 141, 632, self_keys=True, gate=True),
        # the last frame of 16 streams against long 4-bit caches: bound by reading them
        _attn("kv4 16 streams long", "kv4", 16, 1, 1, 20000, 32768, lse=True),
        # own frames and the 4-bit context of the 30 s pair in the fp32 mode
        _attn("kv4 30 s pair f32", "kv4", 2, 750, 750, 576, 576, dtype="f32", self_keys=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cross", "cross", "kv4", "kv4", "append"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    head_dim = rng.choice([128, 128, 128, 64, 96])
    kv_heads = rng.choice([2, 4, 10, 16])
    if op == "append":
        rows = _log(rng, 1, 25600)
        gather = rng.random() < 0.5
        return _append(None, rows, rows + rng.randint(0, 99) if gather else rows, gather, kv_heads, head_dim, dtype)
    group = rng.choice([1, 1, 2, 4])
    kind = rng.choice(["few", "many", "many"])
    if kind == "few":  # the newest frames of some streams
        q_hi = rng.randint(1, 6)
        q_lo = rng.randint(1, q_hi)
        k_hi = _log(rng, 1, 32768 if op == "kv4" else 8192)
        nseq = _log(rng, 1, 16)
    else:  # utterances
        q_hi = _log(rng, 7, 1500)
        q_lo = _log(rng, 1, q_hi)
        k_hi = _log(rng, 1, 2048)
        nseq = _log(rng, 1, 64)
    k_lo = _log(rng, 1, k_hi)
    self_keys = op == "kv4" and rng.random() < 0.6
    c = _attn(None, op, nseq, q_lo, q_hi, k_lo, k_hi, kv_heads * group, kv_heads, head_dim, dtype, self_keys,
              op == "cross" and rng.random() < 0.4, rng.random() < 0.5, rng.random() < 0.5)
    # no dearer than the largest listed cases of its type, padded as the plain form computes it
    most = 1.0e12 if dtype == "bf16" else 1.0e11
    while c["nseq"] > 1 and (4.0 * c["nseq"] * c["heads"] * head_dim * q_hi * (k_hi + (q_hi if self_keys else 0)) > most
                             or c["nseq"] * kv_heads * head_dim * k_hi > 16 * 16 * 128 * 32768):
        c["nseq"] //= 2
    while c["nseq"] * c["heads"] * q_hi * (k_hi + (q_hi if self_keys else 0)) > 1.2e9:
        c["nseq"] = max(1, c["nseq"] // 2)
    return c


def _lens(c):
    """(q_len, k_len) of each sequence: a matter of the case alone."""
    r = random.Random("%(op)s %(nseq)d %(q_lo)d %(q_hi)d %(k_lo)d %(k_hi)d" % c)
    q = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["nseq"])]
    k = [r.randint(c["k_lo"], c["k_hi"]) for _ in range(c["nseq"])]
    return q, k


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _quantise(x):
    """x [rows, heads, head_dim] -> codes [heads, rows, head_dim / 2] (value + 8, even index in the low nibble) and
    scales [heads, rows, groups] of the 4-bit cache.  A scale is the smallest number of 5 significant bits that is at
    least max|x| / 7 of its group; the quotients are taken in 64 bits, where no border is missed."""
    x = x.double().transpose(0, 1)
    h, n, d = x.shape
    pad = -d % GROUP
    g = torch.nn.functional.pad(x, (0, pad)).reshape(h, n, -1, GROUP)
    amax = g.abs().amax(-1)
    frac, exp = torch.frexp(amax / 7)
    s = torch.ldexp(torch.ceil(frac * 32), exp - 5).clamp(max=S_MAX)
    s = torch.where(amax < 2.0 ** -100, torch.zeros_like(s), s)
    c = torch.floor(g.abs() / s.unsqueeze(-1) + 0.5).clamp(max=7) * torch.sign(g)
    c = torch.where(s.unsqueeze(-1) == 0, torch.zeros_like(c), c)
    u = (c.reshape(h, n, d + pad)[..., :d] + 8).to(torch.uint8)
    return (u[..., 0::2] | (u[..., 1::2] << 4)).contiguous(), s.to(torch.bfloat16)


def _values(codes, scales, dtype):
    """The numbers that codes and scales stand for, [heads, rows, head_dim]."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    d = u.shape[-1]
    s = scales.to(dtype).repeat_interleave(GROUP, -1)[..., :d]
    return (u.to(dtype) - 8) * s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    hkv, d = case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    if case["op"] == "kv4_append":
        n, src = case["rows"], case["src_rows"]
        s = {"case": case, "k": normal(src, hkv, d), "v": normal(src, hkv, d), "src_rows": None}
        if case["gather"]:  # the rows that the source's mask leaves, in order
            keep = torch.randperm(src, device="cuda", generator=g)[:n].sort().values
            s["src_rows"] = keep.to(torch.int32)
        s["cache"] = [torch.empty(hkv, n, d // 2, dtype=torch.uint8, device="cuda"),
                      torch.empty(hkv, n, -(-d // GROUP), dtype=torch.bfloat16, device="cuda"),
                      torch.empty(hkv, n, d // 2, dtype=torch.uint8, device="cuda"),
                      torch.empty(hkv, n, -(-d // GROUP), dtype=torch.bfloat16, device="cuda")]
        return s
    h = case["heads"]
    q_len, k_len = _lens(case)
    table, qs, ks = [], 0, 0
    for a, b in zip(q_len, k_len):
        table.append([qs, a, ks, b])
        qs, ks = qs + a, ks + b
    s = {"case": case, "seqs": torch.tensor(table, dtype=torch.int32, device="cuda"), "max_q": max(q_len),
         "max_k": max(k_len), "q": normal(qs, h, d), "k": None, "v": None, "k_self": None, "v_self": None,
         "mask": None, "gate": None, "cache": None}
    if case["op"] == "cross":
        s["k"], s["v"] = normal(ks, hkv, d), normal(ks, hkv, d)
    else:
        s["cache"] = []
        for _ in "kv":
            parts = [_quantise(torch.randn(min(16384, ks - r), hkv, d, device="cuda", generator=g))
                     for r in range(0, ks, 16384)]
            s["cache"] += [torch.cat([p[0] for p in parts], 1), torch.cat([p[1] for p in parts], 1)]
    if case["self_keys"]:
        s["k_self"], s["v_self"] = normal(qs, hkv, d), normal(qs, hkv, d)
    if case["mask"]:  # the last part of some states is padding
        s["mask"] = (torch.rand(ks, device="cuda", generator=g) < 0.9).to(torch.uint8)
    if case["gate"]:
        s["gate"] = torch.sigmoid(torch.randn(qs, h, d, device="cuda", generator=g)).to(dt)
    return s


# ---------------------------------------------------------------------------
# Passes
# ---------------------------------------------------------------------------

def run(state):
    if state["case"]["op"] == "kv4_append":
        return _run_append(state)
    return _run_own(state) if own else _run_plain(state)


def _run_append(state):
    kc, ks, vc, vs = state["cache"]
    if own:
        irt = _pkg()
        cache = irt.Kv4Cache.from_buffers(kc, ks, vc, vs)
        irt.kv4_append(cache, state["k"], state["v"], src_rows=state["src_rows"])
        k, v = irt.kv4_read(cache, dtype=state["k"].dtype)
        return {"k": k, "v": v}
    r = {}
    for name, x, codes, scales in (("k", state["k"], kc, ks), ("v", state["v"], vc, vs)):
        if state["src_rows"] is not None:
            x = x[state["src_rows"].long()]
        c, s = _quantise(x)
        codes.copy_(c)
        scales.copy_(s)
        r[name] = _values(codes, scales, torch.float32).transpose(0, 1).to(x.dtype).contiguous()
    return r


def _run_own(state):
    irt, case = _pkg(), state["case"]
    more = {"gate": state["gate"], "return_lse": case["lse"]}
    if case["op"] == "cross":
        r = irt.cross_attention(state["q"], state["k"], state["v"], state["seqs"], state["max_q"], state["max_k"],
                                key_mask=state["mask"], **more)
    else:
        r = irt.kv4_attention(state["q"], irt.Kv4Cache.from_buffers(*state["cache"]), state["seqs"], state["max_q"],
                              state["max_k"], k_self=state["k_self"], v_self=state["v_self"], **more)
    return {"out": r[0], "lse": r[1]} if case["lse"] else {"out": r}


def _run_plain(state):
    case, t = state["case"], state["seqs"].long()
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    n, mq, mk = t.shape[0], state["max_q"], state["max_k"]

    def rows(start, length, most):
        """Rows of a packed tensor that fill [n, most], and which of them are a sequence's own."""
        at = torch.arange(most, device="cuda")
        ok = at < length[:, None]
        return torch.where(ok, start[:, None] + at, 0), ok

    qi, q_ok = rows(t[:, 0], t[:, 1], mq)
    ki, k_ok = rows(t[:, 2], t[:, 3], mk)
    if state["mask"] is not None:
        k_ok = k_ok & (state["mask"][ki] != 0)
    if state["cache"] is None:
        k, v = state["k"][ki].float(), state["v"][ki].float()
    else:
        kc, ks, vc, vs = state["cache"]
        k = _values(kc[:, ki], ks[:, ki], torch.float32).permute(1, 2, 0, 3)
        v = _values(vc[:, ki], vs[:, ki], torch.float32).permute(1, 2, 0, 3)
    if state["k_self"] is not None:
        k = torch.cat([state["k_self"][qi].float(), k], 1)
        v = torch.cat([state["v_self"][qi].float(), v], 1)
        k_ok = torch.cat([q_ok, k_ok], 1)
    q = state["q"][qi].float().reshape(n, mq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))  # [n, hkv, group * mq, keys]
    scores = torch.where(k_ok[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, h, mq, d).transpose(1, 2)[q_ok]  # [q_rows, heads, head_dim]
    if state["gate"] is not None:
        out = out * state["gate"].float()
    r = {"out": out.to(state["q"].dtype)}
    if case["lse"]:
        r["lse"] = (top + torch.log(total)).reshape(n, h, mq).transpose(1, 2)[q_ok]
    return r


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    hkv, d = case["kv_heads"], case["head_dim"]
    row4 = 2 * hkv * (d // 2 + 2 * -(-d // GROUP))  # one row's K and V in the 4-bit cache
    if case["op"] == "kv4_append":
        # values in, the cache written, its values out
        return {"bytes": case["rows"] * (2 * 2 * hkv * d * size + row4), "flops": case["rows"] * 2 * hkv * d * 4}
    q_len, k_len = _lens(case)
    h, nq, nk = case["heads"], sum(q_len), sum(k_len)
    pairs = sum(a * (b + (a if case["self_keys"] else 0)) for a, b in zip(q_len, k_len))
    b = nq * h * d * size * (3 if case["gate"] else 2) + (nq * h * 4 if case["lse"] else 0)
    b += nk * (row4 if case["op"] == "kv4" else 2 * hkv * d * size) + (nk if case["mask"] else 0)
    b += nq * 2 * hkv * d * size if case["self_keys"] else 0
    return {"bytes": b, "flops": 4 * h * d * pairs}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------

def _exact_cache(x):
    """What the 4-bit cache holds of x [rows, heads, head_dim]."""
    x = x.double()
    out = torch.zeros_like(x)
    for lo in range(0, x.shape[-1], GROUP):
        part = x[..., lo:lo + GROUP]
        amax = part.abs().max(-1, keepdim=True).values
        small = amax < 2.0 ** -100
        want = torch.where(small, 1.0, amax / 7)
        step = torch.exp2(torch.floor(torch.log2(want)) - 4)  # 5 significant bits: 16 to 31 steps
        step = torch.where(want >= 32 * step, 2 * step, torch.where(want < 16 * step, step / 2, step))
        s = torch.minimum(torch.ceil(want / step) * step, torch.full_like(want, S_MAX))
        level = torch.trunc(part.abs() / s + 0.5).clamp(max=7)
        out[..., lo:lo + GROUP] = torch.where(small, 0.0, torch.copysign(level, part) * s)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "kv4_append":
        pick = slice(None) if s["src_rows"] is None else s["src_rows"].long()
        return {"k": _exact_cache(s["k"][pick]), "v": _exact_cache(s["v"][pick])}
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for qs, ql, ks, kl in s["seqs"].tolist():
        if case["op"] == "cross":
            k, v = (s[x][ks:ks + kl].double().transpose(0, 1) for x in "kv")  # [hkv, keys, d]
        else:
            c = s["cache"]
            k = _values(c[0][:, ks:ks + kl], c[1][:, ks:ks + kl], torch.float64)
            v = _values(c[2][:, ks:ks + kl], c[3][:, ks:ks + kl], torch.float64)
        if s["mask"] is not None:
            keep = s["mask"][ks:ks + kl].bool()
            k, v = k[:, keep], v[:, keep]
        if s["k_self"] is not None:
            k = torch.cat([k, s["k_self"][qs:qs + ql].double().transpose(0, 1)], 1)
            v = torch.cat([v, s["v_self"][qs:qs + ql].double().transpose(0, 1)], 1)
        for j in range(h):
            if k.shape[1] == 0:
                lse[qs:qs + ql, j] = -math.inf
                continue
            x = (s["q"][qs:qs + ql, j].double() @ k[j // (h // hkv)].T) / math.sqrt(d)
            lse[qs:qs + ql, j] = torch.logsumexp(x, -1)
            out[qs:qs + ql, j] = torch.softmax(x, -1) @ v[j // (h // hkv)]
    if s["gate"] is not None:
        out = out * s["gate"].double()
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
