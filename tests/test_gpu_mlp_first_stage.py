"""The fused encoder MLP kernel with the output projection in front at hidden size 64, whose first stage is only four steps long, and the engine's
mxfp4 / beam-search paths on the encoder that users get (that kernel, also at the micro architecture): same call, same bits."""
import numpy as np
import pytest

import test_gpu_parity as tp
from moonshine_amd.synth import make_audio
from oracle import moonshine_ref as ref
# the tests of these paths once more, without the switch that keeps the fused kernel out of them
from test_gpu_beam_mxfp4 import (test_beam_search_is_the_search_over_the_engines_logits,  # noqa: F401
                                 test_beam_width_one_is_greedy_and_wider_finds_no_worse, test_beams_of_real_shapes_in_flight_and_profiled,
                                 test_mxfp4_logits_against_the_oracle_on_the_same_values, test_mxfp4_switches_and_refusals, test_transcriber_options,
                                 test_uniform_kernels_give_a_clip_the_same_bits_in_any_batch)
from test_gpu_mlp import _run_o

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("F, R", [(256, 40), (32, 5), (64, 300), (256, 4000)])
def test_block_of_hidden_size_64_is_the_same_every_time(F, R):
    D = 64
    rng = np.random.default_rng(F + R)
    w1 = (rng.standard_normal((F, D)) / np.sqrt(D)).astype(np.float32)
    w2 = (rng.standard_normal((D, F)) / np.sqrt(F)).astype(np.float32)
    wo = (rng.standard_normal((D, D)) / np.sqrt(D)).astype(np.float32)
    b1, b2 = (rng.standard_normal(n).astype(np.float32) * np.float32(0.1) for n in (F, D))
    g = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    h, ao = rng.standard_normal((R, D)).astype(np.float32) * 2, rng.standard_normal((R, D)).astype(np.float32)
    first = _run_o(h, w1, g, b1, w2, b2, ao, wo)
    u = ao.view(np.uint32)
    h1 = h + ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).view(np.float32) @ wo.T
    want = h1 + ref.gelu(ref.layer_norm_nobias(h1, g) @ w1.T + b1) @ w2.T + b2
    err = first - want
    assert float(np.sqrt((err ** 2).mean()) / np.sqrt(((want - h) ** 2).mean())) <= 6e-3 and float(np.abs(err).max()) <= 8e-2
    for _ in range(20):
        np.testing.assert_array_equal(_run_o(h, w1, g, b1, w2, b2, ao, wo), first)


def test_fresh_engines_encode_alike(tmp_path_factory):
    """The first encode of an engine, right behind the allocations of its decode, under the kernel set that takes the fused block for every call."""
    clips = [make_audio(70 + i, 9000 + 4000 * i) for i in range(5)]
    seen = []
    for _ in range(24):
        e, w, cfg = tp._engine(tmp_path_factory, "micro", 0)
        e.set_uniform_kernels(True)
        e.set_keep_encoder_output(True)
        e.encode(clips)
        toks, _ = e.decode(forced_steps=6)
        seen.append(([e.encoder_output(i) for i in range(len(clips))], [list(t) for t in toks]))
        e.close()
    for frames, toks in seen[1:]:
        assert toks == seen[0][1]
        for a, b in zip(frames, seen[0][0]):
            np.testing.assert_array_equal(a, b)
