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
