"""Bounded waits of the attention operators and of the engine's attention over the 4-bit context cache that run out: each
side reports its own and nobody else's.

The waits are those of a probe kernel on a barrier that nothing arrives on, with the limit shortened from 4 s to 50 ms
(no GPU fault, no trap); the test-hook library holds the operators and the engine beside the probe.
"""

import ctypes

import numpy as np
import pytest

from test_gpu_kernels import dev, hooks  # noqa: F401  (fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LIMIT_NS = 50_000_000
U64 = ctypes.POINTER(ctypes.c_ulonglong)


@pytest.fixture()
def probe(pkg, monkeypatch):
    """The package on the test-hook library, and that library."""
    L = hooks()
    for name, (res, args) in pkg._SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    L.irtt_attention_wait_probe.argtypes = [ctypes.c_ulonglong, ctypes.c_int, U64]
    L.irtt_sample_after_expired_wait.argtypes = ([ctypes.c_char_p, ctypes.c_int] + [ctypes.c_void_p] * 2 +
                                                 [ctypes.c_ulonglong] + [ctypes.c_void_p] * 3)
    pkg.lib()
    monkeypatch.setattr(pkg, "_lib", L)
    import irodori_b200.ops as ops
    monkeypatch.setattr(ops, "lib", lambda: L)
    yield L
    L.irt_attention_check(0)


def expire(L, waits=1):
    ns = ctypes.c_ulonglong(0)
    assert L.irtt_attention_wait_probe(LIMIT_NS, waits, ctypes.byref(ns)) == 0, L.irtt_last_error().decode()
    return ns.value


def sampling(pkg, synth, ckpt_dir, name):
    ck = ckpt_dir / f"{name}.safetensors"
    synth.make_dit_checkpoint(str(ck), synth.SMALL_CONFIG, seed=19, init="full")
    r = synth.make_request(synth.SMALL_CONFIG, 1, 20, 12, 48, seed=3)
    req = pkg.SamplingRequest(text_ids=r["text_ids"], text_mask=r["text_mask"], sequence_length=48,
                              ref_latent=r["ref_latent"], ref_mask=r["ref_mask"], initial_noise=r["initial_noise"])
    return ck, req, pkg.SamplerParams(num_steps=2)


def test_the_operators_waits_run_out_report_once_and_clear(pkg, dev, probe):  # noqa: F811
    pkg.attention_check(0)
    ns = expire(probe, waits=8)
    assert LIMIT_NS <= ns < 2 * LIMIT_NS  # one limit for the first wait, none for the others
    with pytest.raises(pkg.IrodoriError) as ei:
        pkg.attention_check(0)
    assert ei.value.kind == "Cuda" and "bounded wait" in str(ei.value)
    pkg.attention_check(0)


@pytest.mark.parametrize("mode", ["native", "4bit"])
def test_sampling_leaves_the_operators_report_alone(pkg, dev, synth, ckpt_dir, probe, mode):  # noqa: F811
    """An expired wait of an operator is no fault of an engine's request, and its report stays for its caller."""
    ck, req, params = sampling(pkg, synth, ckpt_dir, "waits_" + mode)
    eng = pkg.InferenceBuilder(0).load_weights(str(ck)).with_sampling(params).with_context_cache(mode).build()
    want = eng.sample(req)
    expire(probe)
    got = eng.sample(req)
    assert np.linalg.norm(got - want) <= 2e-2 * np.linalg.norm(want)  # two runs of the bf16 engine, each within 1e-2
    with pytest.raises(pkg.IrodoriError):
        pkg.attention_check(0)
    pkg.attention_check(0)


@pytest.mark.parametrize("ql,n", [(1, 1), (70, 40)])  # keys shared by a cluster, and not
@pytest.mark.parametrize("four_bit", [False, True])
def test_a_captured_call_after_an_expired_wait(pkg, dev, probe, four_bit, ql, n):  # noqa: F811
    """Its kernels load nothing and give up at once, not after 4 s a wait, and the report stays.  After the check the same
    graph gives the attention again."""
    h, hd, nk = 4, 128, 700
    g = torch.Generator(device=dev).manual_seed(5)
    q, gate = torch.randn(2, n * ql, h, hd, device=dev, generator=g).to(torch.bfloat16).unbind(0)
    k, v = torch.randn(2, nk, h, hd, device=dev, generator=g).to(torch.bfloat16).unbind(0)
    tab = pkg.attention_table([ql] * n, [nk] * n, [0] * n)
    cache, out = pkg.Kv4Cache(nk, h, hd), torch.zeros_like(q)
    pkg.kv4_append(cache, k, v)

    def call():
        if four_bit:
            pkg.kv4_attention(q, cache, tab, ql, nk, k_self=q, v_self=gate, gate=gate, out=out)
        else:
            pkg.cross_attention(q, k, v, tab, ql, nk, gate=gate, out=out)

    call()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    expire(probe)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    graph.replay()
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 1000
    with pytest.raises(pkg.IrodoriError):
        pkg.attention_check(0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and want.abs().sum() > 0
    pkg.attention_check(0)


def test_the_engine_reports_its_own(pkg, dev, synth, ckpt_dir, probe):  # noqa: F811
    """A wait of the engine's that has run out fails that request and no other, and is no operator's report."""
    ck, req, params = sampling(pkg, synth, ckpt_dir, "waits_engine")
    keep = [np.ascontiguousarray(np.asarray(x), dtype=t) for x, t in
            ((req.text_ids, np.int32), (req.text_mask, np.uint8), (req.ref_latent, np.float32),
             (req.ref_mask, np.uint8), (req.initial_noise, np.float32))]
    ids, tm, ref, rm, noise = keep
    r, sp = pkg._Request(), params._to_c()
    r.batch, r.text_len, r.text_ids, r.text_mask = 1, ids.shape[1], ids.ctypes.data, tm.ctypes.data
    r.ref_len, r.ref_dim, r.ref_latent, r.ref_mask = ref.shape[1], ref.shape[2], ref.ctypes.data, rm.ctypes.data
    r.sequence_length, r.initial_noise, r.memory = 48, noise.ctypes.data, pkg.MEM_HOST
    first, last = np.zeros_like(noise), np.zeros_like(noise)
    statuses = (ctypes.c_int * 3)()
    rc = probe.irtt_sample_after_expired_wait(str(ck).encode(), 0, ctypes.byref(sp), ctypes.byref(r), LIMIT_NS, statuses,
                                              first.ctypes.data, last.ctypes.data)
    message = probe.irtt_last_error().decode()
    assert rc == 0, message
    assert list(statuses) == [0, 20, 0] and "4-bit context cache" in message
    assert np.isfinite(first).all() and np.linalg.norm(last - first) <= 2e-2 * np.linalg.norm(first)
    pkg.attention_check(0)


@pytest.mark.parametrize("four_bit", [False, True])
def test_calls_after_an_expired_wait(pkg, dev, probe, four_bit):  # noqa: F811
    """No call returns success with outputs that mean nothing: they are refused, without a wait for the GPU and inside
    a capture too, until the check has reported the wait."""
    h, hd, nk, ql = 2, 128, 90, 20
    q = torch.randn(ql, h, hd, device=dev).to(torch.bfloat16)
    k, v = torch.randn(2, nk, h, hd, device=dev).to(torch.bfloat16).unbind(0)
    tab, cache, out = pkg.attention_table([ql], [nk]), pkg.Kv4Cache(nk, h, hd), torch.full_like(q, 3.0)

    def call():
        if four_bit:
            return pkg.kv4_attention(q, cache, tab, ql, nk, out=out)
        return pkg.cross_attention(q, k, v, tab, ql, nk, out=out)

    pkg.kv4_append(cache, k, v)
    want = call().clone()
    expire(probe)
    out.fill_(3.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            with pytest.raises(pkg.IrodoriError) as ei:
                call()
            assert ei.value.kind == "Cuda" and "irt_attention_check" in str(ei.value)
        again = q * 1  # the capture goes on
    with pytest.raises(pkg.IrodoriError):
        call()
    pkg.kv4_append(cache, k, v)  # no waits inside: not refused
    pkg.kv4_read(cache)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, q) and (out == 3).all()
    with pytest.raises(pkg.IrodoriError) as ei:
        pkg.attention_check(0)
    assert ei.value.kind == "Cuda" and "bounded wait" in str(ei.value)
    assert torch.equal(call(), want)
    pkg.attention_check(0)
