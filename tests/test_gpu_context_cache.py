"""The engine's 4-bit context cache against the CPU oracle whose context K and
V are replaced by what the cache's format holds of them.

f32 engine: within 1e-4 relative L2, as everywhere.  bf16 engine: the cache is
filled from bf16 rows, so a value near a border between two codes may fall on
the other side: its bf16 rounding moves x by at most 2^-8 |x|, 0.005 of a step
on average (|x| is about 2.6 steps), so about 0.5 % of the values are off by a
step, an rms of sqrt(12 * 0.005) = 0.25 of the rounding error that the format
makes anyway.  What that error does to the latents is the distance d between
the oracle with and without the format; twice 0.25 d is allowed on top of the
bf16 engine's own 1e-2.
"""

import numpy as np
import pytest
import torch

from test_gpu_ctx_attention import quantised

pytestmark = pytest.mark.gpu


def rel_l2(a, b):
    a, b = np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


class QuantisedKv:
    """A context K/V cache seen through the 4-bit format."""

    def __init__(self, kv):
        self._kv = kv
        self.ctx_k = quantised(kv.ctx_k).to(kv.ctx_k.dtype)
        self.ctx_v = quantised(kv.ctx_v).to(kv.ctx_v.dtype)

    def __getattr__(self, name):
        return getattr(self._kv, name)


def sample_oracle(oracle, monkeypatch, ckpt, req, params, four_bit):
    W = oracle.Weights.load(str(ckpt))
    with monkeypatch.context() as m:
        if four_bit:
            plain = oracle.joint_attention
            m.setattr(oracle, "joint_attention", lambda W, p, h, kv, *a: plain(W, p, h, QuantisedKv(kv), *a))
        with torch.no_grad():
            return oracle.sample_euler_rf_cfg(W, req, params).numpy()


CASES = [
    ("small", "joint", {}),
    ("small", "independent", {}),
    ("small", "independent", dict(scale=1.7, max_layers=1)),  # scaled speaker rows, first layer only
    ("tiny", "alternating", {}),                              # head_dim 8: one group of 8 values a row
]


@pytest.mark.parametrize("size,mode,skv", CASES)
@pytest.mark.parametrize("precision", ["f32", "bf16"])
def test_sampling_over_the_4bit_cache(pkg, oracle, synth, ckpt_dir, monkeypatch, size, mode, skv, precision):
    ck = ckpt_dir / f"ctx_{size}.safetensors"
    cfg = synth.SMALL_CONFIG if size == "small" else synth.TINY_CONFIG
    synth.make_dit_checkpoint(str(ck), cfg, seed=11, init="full")
    S, steps = 90, 3
    r = synth.make_request(cfg, 2, 40, 50, S, seed=5)
    r["text_mask"][1, 30:] = False
    fields = dict(text_ids=r["text_ids"], text_mask=r["text_mask"], sequence_length=S, ref_latent=r["ref_latent"],
                  ref_mask=r["ref_mask"], initial_noise=r["initial_noise"])
    op = oracle.SamplerParams(num_steps=steps, guidance=oracle.GuidanceConfig(mode=mode, scale_text=3.0, scale_speaker=3.0),
                              speaker_kv=oracle.SpeakerKvConfig(**skv) if skv else None)
    want = sample_oracle(oracle, monkeypatch, ck, oracle.SamplingRequest(**fields), op, True)
    native = sample_oracle(oracle, monkeypatch, ck, oracle.SamplingRequest(**fields), op, False)
    params = pkg.SamplerParams(num_steps=steps, guidance=pkg.GuidanceConfig(mode=mode, scale_text=3.0, scale_speaker=3.0),
                               speaker_kv=pkg.SpeakerKvConfig(**skv) if skv else None)
    eng = (pkg.InferenceBuilder(0).load_weights(str(ck), precision=precision).with_sampling(params)
           .with_context_cache("4bit").build())
    d = rel_l2(want, native)
    own = 1e-4 if precision == "f32" else 1e-2
    tol = own if precision == "f32" else own + 0.5 * d

    def run():
        return eng.sample(pkg.SamplingRequest(**fields))

    # the first request runs eagerly, the next ones from CUDA graphs.  (Runs are compared with the oracle, not with one
    # another: the bf16 residual GEMMs add their K-splits in any order.)
    for _ in range(3):
        err = rel_l2(run(), want)
        assert err < tol, (err, tol, d)
    # the native cache is back when asked for, and the 4-bit one after it
    eng.with_context_cache("native")
    err = rel_l2(run(), native)
    assert err < own, err
    eng.with_context_cache("4bit")
    err = rel_l2(run(), want)
    assert err < tol, (err, tol, d)


def test_no_context_rows_and_refusals(pkg, synth, ckpt_dir):
    """A request whose text is all masked has no context rows at all."""
    ck = ckpt_dir / "ctx_empty.safetensors"
    cfg = synth.SMALL_CONFIG
    synth.make_dit_checkpoint(str(ck), cfg, seed=12, init="full")
    S = 64
    r = synth.make_request(cfg, 1, 8, 4, S, seed=6)
    req = pkg.SamplingRequest(text_ids=r["text_ids"], text_mask=np.zeros_like(np.asarray(r["text_mask"])),
                              sequence_length=S, initial_noise=r["initial_noise"])
    eng = pkg.InferenceBuilder(0).load_weights(str(ck)).with_sampling(pkg.SamplerParams(num_steps=2)).build()
    plain = eng.sample(req)
    err = rel_l2(eng.with_context_cache("4bit").sample(req), plain)
    assert err < 2e-2, err  # two runs of the bf16 engine, each within 1e-2
    with pytest.raises(pkg.IrodoriError) as ei:
        eng.with_context_cache("8bit")
    assert ei.value.kind == "InvalidArgument"
