"""What the engine's context cache takes of the GPU's memory when its mode changes."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_changed_mode_gives_the_other_caches_memory_back(pkg, synth, ckpt_dir):
    """The context of the batch takes two layers x (K and V) x rows x 256 values: 4 bytes each natively, 4.5 bits over
    4 bits beside one native layer.  An engine that changes its mode holds what one holds that never had the other,
    to the allocator's granularity (2 MiB a buffer; four buffers are replaced)."""
    ck = ckpt_dir / "ctx_memory.safetensors"
    cfg = synth.SMALL_CONFIG
    synth.make_dit_checkpoint(str(ck), cfg, seed=13, init="full")
    B, T, S = 32, 1024, 16
    rows = 2 * B * T
    r = synth.make_request(cfg, B, T, T, S, seed=7)
    req = pkg.SamplingRequest(text_ids=r["text_ids"], text_mask=np.ones_like(np.asarray(r["text_mask"])),
                              sequence_length=S, ref_latent=r["ref_latent"], ref_mask=np.ones_like(np.asarray(r["ref_mask"])),
                              initial_noise=r["initial_noise"])
    eng = (pkg.InferenceBuilder(0).load_weights(str(ck), precision="f32")
           .with_sampling(pkg.SamplerParams(num_steps=3)).with_context_cache("native").build())

    def held():
        torch.cuda.synchronize()
        free, total = torch.cuda.mem_get_info(0)
        return total - free

    def sampled(mode):
        eng.with_context_cache(mode).sample(req)
        out = eng.sample(req)  # a second one: graphs too
        return out, held()

    native = 2 * 2 * rows * 256 * 4
    four = native // 2 + 2 * 2 * rows * (256 // 2 + 2 * 256 // 32)
    slack = 16 << 20
    first, a = sampled("native")
    _, b = sampled("4bit")
    again, c = sampled("native")
    _, d = sampled("4bit")
    print(f"native {native >> 20} MiB, 4-bit {four >> 20} MiB, held {[(x - a) >> 20 for x in (a, b, c, d)]} MiB beside native")
    assert native - four > 2 * slack
    assert b <= a - (native - four) + slack
    assert abs(c - a) <= slack and abs(d - b) <= slack
    assert np.linalg.norm(again - first) <= 1e-4 * np.linalg.norm(first)
