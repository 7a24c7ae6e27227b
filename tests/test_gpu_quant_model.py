"""The bf16 decoder over caches in 4 and 8 bits: prompt and cached steps against the stacked layer oracle, whose cached rows are what a
quantised cache holds; the graphed step; generation from a model folder's options."""
import numpy as np
import pytest
import torch

from oracle import model_oracle
from oracle import quant_cache_oracle as qo
from tests.test_gpu_model import _check, _params

pytestmark = pytest.mark.gpu


def _hold(bits, heads):
    def hold(rows, which):
        by_head = rows.reshape(len(rows), heads, -1)
        return qo.held(by_head, bits[0 if which == "k" else 1]).reshape(rows.shape).astype(np.float32)

    return hold


@pytest.mark.parametrize("bits", [(4, 4), (8, 4), (8, 8)])
@pytest.mark.parametrize("ragged", [False, True])
def test_decoder_over_a_quantised_cache(pkg, bits, ragged):
    """The tolerance is that of the decoder over bf16 caches (6e-2 on logits).  What comes on top is a code that falls on the other side of a
    border because the device's row differs from the oracle's in bf16's last bit: one step, at most 1 / 7 of a group's largest element, of one token in
    48 or more."""
    from llm_experiments_b200 import model

    gpu = pkg.gpu
    ctx = gpu.context_create(0)
    cfg = model.DecoderConfig(vocab_size=512, context_size=96, embedding_dim=256, n_heads=2, n_layers=2)
    params = _params(cfg, model, seed=3)
    weights = model.weights_from_numpy(ctx, cfg, params)
    B, N, steps = 3, 48, 4
    hold = _hold(bits, cfg.n_heads)
    state = model.decoder_state_create(ctx, cfg, weights, batch_size=B, ragged=ragged, kv_bits=bits)
    prompt = np.random.default_rng(1).integers(0, cfg.vocab_size, size=B * N).astype(np.int32)
    ids = gpu.gpu_buffer_1d_create(ctx, B * N, torch.from_numpy(prompt), dtype=torch.int32)
    nxt = gpu.gpu_buffer_1d_create(ctx, B, dtype=torch.int32)
    ctx.config.check_device_status = True
    for _ in range(2):  # a second prompt starts the caches over
        gpu.batch_begin(ctx)
        model.prefill(ctx, state, ids, N, nxt)
        gpu.batch_commit(ctx)
    want, cache = model_oracle.prefill(params, prompt, B, N, cfg.n_heads, hold)
    got_next = nxt.buffer.cpu().numpy()
    _check(state.logits.buffer, want, got_next, "prompt")
    for step in range(steps):
        tokens = got_next.copy()
        tok = gpu.gpu_buffer_1d_create(ctx, B, torch.from_numpy(tokens), dtype=torch.int32)
        gpu.batch_begin(ctx)
        model.decode_step(ctx, state, tok, nxt)
        gpu.batch_commit(ctx)
        want = model_oracle.decode_step(params, tokens, cache, cfg.n_heads, hold)
        got_next = nxt.buffer.cpu().numpy()
        _check(state.logits.buffer, want, got_next, f"step {step}")
        assert all(c.current_len == N + step + 1 for c in state.caches)


def test_graphed_step_over_a_quantised_cache(pkg):
    from llm_experiments_b200 import model

    gpu = pkg.gpu
    ctx = gpu.context_create(0)
    cfg = model.DecoderConfig(vocab_size=512, context_size=96, embedding_dim=256, n_heads=2, n_layers=2)
    weights = model.weights_from_numpy(ctx, cfg, _params(cfg, model, seed=9))
    B, N, steps, lens = 3, 32, 5, [32, 7, 19]
    prompt = np.random.default_rng(4).integers(0, cfg.vocab_size, size=B * N).astype(np.int32)
    runs = []
    for graphed in (False, True):
        state = model.decoder_state_create(ctx, cfg, weights, batch_size=B, ragged=True, kv_bits=(8, 4))
        ids = gpu.gpu_buffer_1d_create(ctx, B * N, torch.from_numpy(prompt), dtype=torch.int32)
        nxt = gpu.gpu_buffer_1d_create(ctx, B, dtype=torch.int32)
        gpu.batch_begin(ctx)
        model.prefill(ctx, state, ids, N, nxt)
        gpu.batch_commit(ctx)
        for c in state.caches:
            gpu.quant_cache_set_lengths(c, lens)
        step = model.GraphedDecodeStep(ctx, state) if graphed else None
        tok = step.token_ids if graphed else gpu.gpu_buffer_1d_create(ctx, B, dtype=torch.int32)
        if graphed:
            step.capture()
            assert state.caches[0].seq_lens.tolist() == lens
        logits = []
        for i in range(steps):
            tok.buffer.copy_(torch.from_numpy(np.random.default_rng(10 + i).integers(0, cfg.vocab_size, size=B).astype(np.int32)))
            if graphed:
                step.step()
            else:
                gpu.batch_begin(ctx)
                model.decode_step(ctx, state, tok, nxt)
                gpu.batch_commit(ctx)
            logits.append(state.logits.buffer.float().cpu())
        assert state.caches[-1].seq_lens.tolist() == [n + steps for n in lens]
        runs.append(logits)
    for a, b in zip(*runs):  # (the captured launch is cut for the cache's capacity: fp32 sums in another order)
        assert float((a - b).abs().max()) <= 2e-2


def test_generation_over_a_quantised_cache(pkg):
    from llm_experiments_b200 import generate, model

    ctx = pkg.gpu.context_create(0)
    cfg = model.DecoderConfig(vocab_size=512, context_size=64, embedding_dim=256, n_heads=2, n_layers=2)
    dec = model.CachedDecoder(ctx, cfg, model.weights_from_numpy(ctx, cfg, _params(cfg, model, seed=5)), kv_bits=(8, 8))
    prompt = [int(t) for t in np.random.default_rng(2).integers(0, 512, size=9)]
    first = generate.generate_text(dec, prompt, max_tokens=6, temperature=0.0)
    assert first[:9] == prompt and len(first) == 15 and generate.generate_text(dec, prompt, max_tokens=6, temperature=0.0) == first


def test_generation_from_a_model_folder(pkg, tmp_path):
    """``kv_bits`` of ``config.json``: the same tokens as of a decoder made with them, over caches of those bits."""
    import json

    from llm_experiments_b200 import checkpoint, generate, model

    ctx = pkg.gpu.context_create(0)
    cfg = model.DecoderConfig(vocab_size=512, context_size=64, embedding_dim=256, n_heads=2, n_layers=2)
    params = _params(cfg, model, seed=5)
    tensors = {k: params[k] for k in ("embedding", "out_proj", "lnf_gamma", "lnf_beta")}
    tensors.update({f"layers.{i}.{k}": x for i, layer in enumerate(params["layers"]) for k, x in layer.items()})
    checkpoint.write_safetensors(tmp_path / "model.safetensors", {k: torch.from_numpy(x).to(torch.bfloat16) for k, x in tensors.items()})
    (tmp_path / "config.json").write_text(json.dumps(dict(architecture="GPTDecoder", vocab_size=512, context_size=64, embedding_dim=256, n_heads=2, n_layers=2,
                                                          kv_bits=[8, 4])))
    loaded = pkg.gpu.load_model(ctx, tmp_path)
    assert all(isinstance(c, pkg.gpu.QuantKVCache) and (c.k_bits, c.v_bits) == (8, 4) for c in loaded.state.caches)
    prompt = [int(t) for t in np.random.default_rng(2).integers(0, 512, size=9)]
    made = model.CachedDecoder(ctx, cfg, model.weights_from_numpy(ctx, cfg, params), kv_bits=(8, 4))
    got = generate.generate_text(loaded, prompt, max_tokens=6, temperature=0.0)
    assert len(got) == 15 and got == generate.generate_text(made, prompt, max_tokens=6, temperature=0.0)
