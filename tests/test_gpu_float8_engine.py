"""The engine with its layers' matrices in 8 bits against the plain implementation on the same, dequantised, weights.

What is left between the two is the rounding of what the products read: a number to e4m3 is off by at most 2^-4 of it, uniformly over a step at the
worst, 2^-4 / sqrt(3) in the mean square; four products a layer read such rows, and the errors of different products have nothing to do with each
other, so the logits of L layers are off by at most 2^-4 / sqrt(3) * sqrt(4 L) of their norm (a branch's error is that of what it reads, weighted
with the branch's share of the stream, which is at most one)."""
import os
import subprocess

import numpy as np
import pytest
import torch

import helpers as H
import plain_model as pm

pytestmark = pytest.mark.gpu


def bound(which):
    return 2.0 ** -4 / 3 ** 0.5 * (4 * H.TINY[which]["num_hidden_layers"]) ** 0.5


def engine(d, which, **kw):
    return H.engine_for(d, "bfloat16", H.PAGE_SIZE[which], 512, weights="float8", **kw)


def dequantised(m):
    N, width = m.codes.shape
    s = m.scales.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :width]
    return (m.codes.double() * s.double()).cpu().numpy()


def weights_of(eng, d):
    """The checkpoint's tensors with the layers' matrices as the engine has them."""
    config, weights = pm.load_model_folder(d)
    for i, block in enumerate(eng.model.blocks):
        p, mixer, ff = f"model.layers.{i}.", block.mixer, block.feed_forward
        qkv, gu = dequantised(mixer.w_qkv), dequantised(ff.w_gate_up)
        q, kv = mixer.q_dim, mixer.kv_dim
        if ff.group:
            v = gu.reshape(-1, 2, ff.group, gu.shape[1])
            gate, up = v[:, 0].reshape(-1, gu.shape[1]), v[:, 1].reshape(-1, gu.shape[1])
        else:
            gate, up = gu[:ff.intermediate_size], gu[ff.intermediate_size:]
        for name, t in (("self_attn.q_proj", qkv[:q]), ("self_attn.k_proj", qkv[q:q + kv]), ("self_attn.v_proj", qkv[q + kv:]),
                        ("self_attn.o_proj", dequantised(mixer.w_o)), ("mlp.gate_proj", gate), ("mlp.up_proj", up), ("mlp.down_proj", dequantised(ff.w_down))):
            assert t.shape == weights[p + name + ".weight"].shape
            weights[p + name + ".weight"] = t.astype(np.float32)
    return config, weights


def rows(collected, rid):
    return np.stack([collected[rid][p] for p in sorted(collected[rid])])


@pytest.mark.parametrize("which", list(H.TINY))
def test_whole_in_portions_and_token_by_token(tmp_path, which):
    d = H.make_folder(tmp_path, which)
    eng = engine(d, which)
    toks = H.tokens_for(which, 90, 5)
    want = pm.decoder_forward(*weights_of(eng, d), toks)
    ways = {
        "whole": [([(1, toks, list(range(90)))], [1])],
        "portions": [([(2, toks[a:b], list(range(b - a)))], [2] if b == 90 else []) for a, b in ((0, 40), (40, 57), (57, 90))],
        "tail one by one": [([(3, toks[:70], list(range(70)))], [])] + [([(3, [toks[i]], [0])], [3] if i == 89 else []) for i in range(70, 90)],
    }
    for (what, steps), rid in zip(ways.items(), (1, 2, 3)):
        got = rows(H.run_steps(eng, steps), rid)
        assert got.shape == want.shape and np.isfinite(got).all()
        off = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert off < bound(which), (what, off)
    from aien_sovereign_core_mv_b200 import kernels as K
    assert K.read_wait_errors() == (0, 0, 0, 0)


@pytest.mark.parametrize("which", ["A", "B"])
def test_graphs_and_recorded_steps_change_no_bit(tmp_path, which):
    """Decode steps through captured graphs, and prompt steps re-issued as recorded, against the same steps launched one by one."""
    d = H.make_folder(tmp_path, which)
    toks = {r: H.tokens_for(which, 60, r) for r in (1, 2, 3)}
    got = []
    for kw in (dict(use_cuda_graphs=False, replay_steps=False), dict()):
        eng = engine(d, which, **kw)
        steps = []
        for again in range(3):                           # the same shapes again: recorded, then re-issued
            steps += [([(10 * again + r, t[:33], [32]) for r, t in toks.items()], [])]
            steps += [([(10 * again + r, [t[i]], [0]) for r, t in toks.items()], [10 * again + r for r in toks] if i == 45 else []) for i in range(33, 46)]
        got.append(H.run_steps(eng, steps))
    for rid in got[0]:
        assert np.array_equal(rows(got[0], rid), rows(got[1], rid))


def test_a_larger_layer_with_a_prompt_and_a_batch(tmp_path):
    """Sizes that reach every form of the product: a prompt of 700 tokens (pairs of CTAs and single ones), 20 users, one user."""
    raw = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", num_hidden_layers=2, hidden_size=1024, num_attention_heads=16,
               num_key_value_heads=4, head_dim=128, intermediate_size=2816, vocab_size=512, rope_theta=1000000.0, rms_norm_eps=1e-6,
               tie_word_embeddings=False, max_position_embeddings=2048, hidden_act="silu", attention_bias=False, eos_token_id=0)
    from aien_sovereign_core_mv_b200 import Engine, EngineConfig, write_random_model
    d = str(tmp_path / "m")
    write_random_model(d, raw, 9, None)
    eng = Engine.from_folder(d, EngineConfig(dtype="bfloat16", weights="float8", page_size=16, max_cache_tokens=4096, max_requests=32, max_context=1024))
    rng = np.random.default_rng(4)
    toks = rng.integers(0, 512, 705).tolist()
    got = [np.asarray(eng.step([(1, toks[:700], [0, 350, 699])]).cpu())] + [np.asarray(eng.step([(1, [t], [0])]).cpu()) for t in toks[700:]]
    want = pm.decoder_forward(*weights_of(eng, d), toks)[[0, 350, 699, 700, 701, 702, 703, 704]]
    got = np.concatenate(got)
    lim = 2.0 ** -4 / 3 ** 0.5 * 8 ** 0.5
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < lim
    eng.end_request(1)
    batch = {r: rng.integers(0, 512, 21).tolist() for r in range(2, 22)}
    eng.step([(r, t[:20], []) for r, t in batch.items()])
    got = np.asarray(eng.step([(r, t[20:], [0]) for r, t in batch.items()]).cpu())
    config, weights = weights_of(eng, d)
    want = np.stack([pm.decoder_forward(config, weights, t)[20] for t in batch.values()])
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < lim


def test_command_line(tmp_path):
    d = H.make_folder(tmp_path, "B")
    cmd = [os.path.join(H.ROOT, "bin", "aien-b200"), "generate", "--model-dir", d, "--weights", "float8", "--prompt-ids", "5,6,7,8", "--max-tokens", "5",
           "--temperature", "0", "--stop-token-ids", "", "--json"]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr
    assert len(__import__("json").loads(out.stdout.strip().splitlines()[-1])["tokens"][0]) == 5
    bad = subprocess.run(cmd + ["--dtype", "float32"], capture_output=True, text=True, timeout=600)
    assert bad.returncode == 1 and "bfloat16" in bad.stderr
