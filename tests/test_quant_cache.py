"""Quantised key / value cache without a GPU: the oracle against its definition, and what the operators refuse."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo


@pytest.fixture()
def ctx(pkg):
    gpu = pkg.gpu
    return gpu.GPUContext(device=torch.device("cpu"), config=gpu.GPUConfig(), batch_state=None)


def make(pkg, ctx, **kw):
    base = dict(batch_size=2, max_seq_len=40, n_layers=1, n_kv_heads=2, head_dim=64)
    base.update(kw)
    return pkg.gpu.quant_cache_create(ctx, pkg.gpu.QuantKVCacheConfig(**base))


def two(pkg, rows, cols, dtype=torch.bfloat16):
    return pkg.gpu.GPUBuffer2D(buffer=torch.zeros((rows, cols), dtype=dtype), shape=(rows, cols), size=rows * cols)


# ---- the oracle ----

def test_bfloat16_rounding_is_torch_s():
    x = np.concatenate([np.random.default_rng(0).standard_normal(4096) * 10.0 ** np.random.default_rng(1).integers(-38, 38, 4096),
                        [0.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 3.4e38, 2.0 ** -133, 2.0 ** -134, 1.5 * 2.0 ** -134]]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    np.testing.assert_array_equal(qo.to_bf16(x), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_is_within_half_a_step_and_keeps_the_largest(bits):
    top = 7 if bits == 4 else 127
    x = np.random.default_rng(2).standard_normal((5, 64)) * np.array([1e-30, 1e-3, 1, 100, 1e30])[:, None]
    codes, scales = qo.quantise(x, bits)
    assert np.abs(codes).max() == top and np.all(codes == np.rint(codes))
    step = np.repeat(scales, 32, axis=-1)
    # half a step, and the part of the largest element that the scale's own rounding cuts off (half a step of bfloat16, 2^-8)
    assert np.all(np.abs(codes * step - x) <= step * (0.5 + top * 2.0 ** -8))
    zero, _ = qo.quantise(np.zeros((1, 32)), bits)
    assert not zero.any()
    bad = np.ones((2, 64))
    bad[0, 3], bad[1, 40] = np.inf, np.nan
    back = qo.held(bad, bits)
    assert np.isnan(back[0, :32]).all() and np.isnan(back[1, 32:]).all() and np.isfinite(back[0, 32:]).all()


def test_attention_of_the_oracle_on_hand_made_cases():
    v = np.array([[[1.0, 2.0]], [[3.0, -2.0]], [[5.0, 8.0]]])
    k = np.zeros_like(v)
    q = np.ones((2, 1, 2))
    out, _, _ = qo.attention(q, k, v, 1.0)
    np.testing.assert_allclose(out[0, 0], [2.0, 0.0])      # the first of two queries sees two tokens
    np.testing.assert_allclose(out[1, 0], [3.0, 8.0 / 3])
    out, _, _ = qo.attention(q, k, v, 1.0, window=1)
    np.testing.assert_allclose(out[:, 0], v[1:, 0])
    out, _, _ = qo.attention(np.ones((5, 1, 2)), k, v, 1.0)  # more queries than tokens: the first two see nothing
    assert not out[:2].any() and np.allclose(out[2, 0], v[0, 0])
    out, _, _ = qo.attention(q, k, v, 1.0, slopes=[np.log(2.0)])
    np.testing.assert_allclose(out[0, 0], (v[0, 0] / 2 + v[1, 0]) / 1.5)
    k[0, 0] = [1e4, 1e4]
    out, _, _ = qo.attention(q, k, v, 1.0, softcap=np.log(3.0))
    np.testing.assert_allclose(out[0, 0], (3 * v[0, 0] + v[1, 0]) / 4)


# ---- refusals ----

def test_create_refuses_what_no_kernel_takes(pkg, ctx):
    for field in ("batch_size", "max_seq_len", "n_layers", "n_kv_heads", "head_dim"):
        with pytest.raises(ValueError, match=f"{field} must be > 0, got 0"):
            make(pkg, ctx, **{field: 0})
    with pytest.raises(ValueError, match="head_dim 80"):
        make(pkg, ctx, head_dim=80)
    with pytest.raises(ValueError, match="k_bits"):
        make(pkg, ctx, k_bits=4, v_bits=8)
    with pytest.raises(ValueError, match="dtype"):
        make(pkg, ctx, dtype=torch.float16)
    with pytest.raises(ValueError, match="n_blocks"):
        make(pkg, ctx, block_size=16, n_blocks=5)
    with pytest.raises(ValueError, match="max_seq_len must be at most"):
        make(pkg, ctx, max_seq_len=(1 << 30) + 1)
    with pytest.raises(ValueError, match="block_size"):
        make(pkg, ctx, block_size=-16)


@pytest.mark.parametrize("bits", [(4,), (8, 8, 8), (4, 8), (5, 5)])
def test_a_decoder_refuses_other_bits(pkg, ctx, bits):
    from llm_experiments_b200 import model
    with pytest.raises(ValueError, match="bits"):
        model.decoder_state_create(ctx, model.DecoderConfig(vocab_size=64, context_size=32, embedding_dim=64, n_heads=1, n_layers=1), None, 1, kv_bits=bits)


def test_create_sizes(pkg, ctx):
    c = make(pkg, ctx, head_dim=128, k_bits=8, n_layers=2)
    lay = c.layers[1]
    assert lay.k_codes.shape == (2 * 2 * 40, 128) and lay.v_codes.shape == (160, 64) and lay.k_scales.shape == (160, 4)
    assert make(pkg, ctx, head_dim=96).layers[0].k_scales.shape == (160, 4) and make(pkg, ctx, head_dim=32).layers[0].v_scales.shape == (160, 2)
    paged = make(pkg, ctx, block_size=24, n_blocks=7, ragged=True)
    assert paged.layers[0].k_codes.shape == (7 * 2 * 24, 32) and paged.block_table.tolist() == [[0, 1], [2, 3]] and paged.seq_lens.tolist() == [0, 0]
    pkg.gpu.quant_cache_set_lengths(paged, [3, 40])
    assert paged.current_len == 40 and paged.seq_lens.tolist() == [3, 40]
    with pytest.raises(ValueError):
        pkg.gpu.quant_cache_set_lengths(paged, [3, 41])
    pkg.gpu.quant_cache_reset(paged)
    assert paged.current_len == 0 and paged.seq_lens.tolist() == [0, 0]


def test_update_and_gather_refusals(pkg, ctx):
    gpu, c = pkg.gpu, make(pkg, ctx)
    good = two(pkg, 2, 128)
    with pytest.raises(ValueError, match=r"layer_idx 1 out of range"):
        gpu.quant_cache_update(ctx, c, 1, good, good)
    with pytest.raises(ValueError, match="shape mismatch"):
        gpu.quant_cache_update(ctx, c, 0, good, two(pkg, 2, 64))
    with pytest.raises(ValueError, match="dtype"):
        gpu.quant_cache_update(ctx, c, 0, good, two(pkg, 2, 128, torch.float32))
    with pytest.raises(ValueError, match="tokens"):
        gpu.quant_cache_update(ctx, c, 0, good, good, tokens=0)
    with pytest.raises(ValueError, match="shape mismatch"):
        gpu.quant_cache_update(ctx, c, 0, good, good, tokens=2)
    across = gpu.GPUBuffer2D(buffer=torch.zeros((128, 2), dtype=torch.bfloat16).t(), shape=(2, 128), size=256)
    with pytest.raises(ValueError, match="next to one another"):
        gpu.quant_cache_update(ctx, c, 0, across, good)
    c.current_len = 40
    with pytest.raises(ValueError, match="Cache is full"):
        gpu.quant_cache_update(ctx, c, 0, good, good)
    with pytest.raises(ValueError, match="which"):
        gpu.quant_cache_gather(ctx, c, 0, "q")
    with pytest.raises(ValueError, match="length"):
        gpu.quant_cache_gather(ctx, c, 0, "k", length=0)
    with pytest.raises(RuntimeError, match="batch_begin"):
        c.current_len = 0
        gpu.quant_cache_update(ctx, c, 0, good, good)
    assert c.current_len == 0


def test_attention_refusals(pkg, ctx):
    gpu, c = pkg.gpu, make(pkg, ctx)
    q = two(pkg, 2, 256)

    def refused(text, q=q, out=q, **kw):
        with pytest.raises(ValueError, match=text):
            gpu.attention_with_quant_cache(ctx, c, 0, q, out, **kw)

    refused("Cache is empty")
    c.current_len = 30
    refused("tokens", tokens=0)
    refused("tokens", tokens=65)
    refused("pending", pending=11)
    refused("pending", pending=-1)
    refused("window", window=-1)
    refused("softcap", softcap=-1.0)
    refused("softcap", softcap=float("inf"))
    refused("softcap", softcap=1e-40)
    refused("scale", scale=float("nan"))
    refused("columns", q=two(pkg, 2, 192))
    refused("columns", q=two(pkg, 2, 100))
    refused("shape mismatch", out=two(pkg, 2, 128))
    refused("shape mismatch", tokens=2)
    refused("dtype", q=two(pkg, 2, 256, torch.float32))
    slopes = lambda n, dtype=torch.float32: gpu.GPUBuffer1D(buffer=torch.zeros(n, dtype=dtype), shape=(n,), size=n)  # noqa: E731
    refused("slopes", slopes=slopes(3))
    refused("slopes", slopes=slopes(4, torch.float64))
    with pytest.raises(RuntimeError, match="batch_begin"):
        gpu.attention_with_quant_cache(ctx, c, 0, q, q)


def test_numbers_beyond_float32_are_refused(pkg, ctx):
    gpu, c = pkg.gpu, make(pkg, ctx)
    c.current_len = 30
    q = two(pkg, 2, 256)
    for kw in (dict(softcap=1e300), dict(softcap=3.5e38), dict(scale=1e300), dict(scale=-3.5e38), dict(softcap=float("nan")), dict(scale=float("-inf"))):
        with pytest.raises(ValueError, match="softcap"):
            gpu.attention_with_quant_cache(ctx, c, 0, q, q, **kw)


def test_entry_points_check_before_any_launch(pkg):
    native = pkg._native
    lib, A = native.lib, 0x1000
    fields = dict(k=A, v=A, ks=A, vs=A, table=0, lens=0, len=4, B=1, G=2, D=64, T=8, max_blocks=0, block=0, n_blocks=0, kb=4, vb=4, dt=1)

    def cache(**kw):
        return native.qcache(*{**fields, **kw}.values())

    def write(k=A, ld=128, n=1, **kw):
        return lib.b2kv_qcache_write(cache(**kw), k, ld, A, 128, n, None, None)

    assert write(dt=7) == -3 and write(D=80) == -3 and write(kb=4, vb=8) == -3 and write(kb=2) == -3
    assert write(k=None) == -1 and write(ks=0) == -1 and write(B=0) == -1 and write(n=0) == -1 and write(n=5) == -1 and write(ld=64) == -1
    assert write(T=(1 << 30) + 1) == -3
    assert write(len=-1) == -1 and write(len=8) == -1
    assert write(k=A + 8) == -2 and write(ld=132) == -2 and write(v=A + 4) == -2
    assert write(table=A) == -1 and write(table=A, max_blocks=1, block=4, n_blocks=1) == -1  # a table that does not hold T_max
    read = lambda which=0, out=A, n=1, **kw: lib.b2kv_qcache_read(cache(**kw), which, out, n, 0, 0, None, None)  # noqa: E731
    assert read(which=2) == -1 and read(out=None) == -1 and read(n=0) == -1 and read(out=A + 8) == -2 and read(D=48) == -3

    args = dict(q=A, out=A, slopes=0, ld_q=256, ld_out=256, H=4, m=1, T=4, bias=0, window=0, scale=0.125, cap=0.0)

    def attend(ws=None, nbytes=0, c=None, **kw):
        return lib.b2kv_qcache_attend(cache(**(c or {})), native.qcache_attend_args(*{**args, **kw}.values()), ws, nbytes, None, None)

    assert attend(q=0) == -1 and attend(H=3) == -1 and attend(m=0) == -1 and attend(T=9) == -1 and attend(window=-1) == -1
    assert attend(m=65) == -3 and attend(c=dict(D=80)) == -3
    assert attend(scale=float("nan")) == -1 and attend(cap=-1.0) == -1 and attend(cap=1e-35) == -1 and attend(ld_q=128) == -1
    assert attend(ld_out=260) == -2 and attend(q=A + 2) == -2
    big, long_args = dict(T=1 << 20), dict(T=1 << 20)
    need = lib.b2kv_qcache_attend_workspace_bytes(cache(**big), native.qcache_attend_args(*{**args, **long_args}.values()))
    assert need > 0 and attend(c=big, **long_args) == -4 and attend(ws=A, nbytes=need - 1, c=big, **long_args) == -4
    assert attend(ws=A + 4, nbytes=need, c=big, **long_args) == -2
    assert lib.b2kv_qcache_attend_workspace_bytes(cache(D=80), native.qcache_attend_args(*args.values())) == 0
    assert [lib.b2kv_qcache_scale_row(d) for d in (32, 64, 96, 128, 256, 80, 0)] == [2, 2, 4, 4, 8, 0, 0]
    assert ctypes.sizeof(native.QCache) == 96 and ctypes.sizeof(native.QCacheAttendArgs) == 72


@pytest.mark.parametrize("D,bits,wide", [(128, (8, 4), True), (256, (4, 4), True), (256, (8, 8), True), (256, (8, 4), False)])
def test_columns_that_are_taken_together(pkg, D, bits, wide):
    """Scratch memory tells the tiles apart: results of 16 columns per CTA, or of 8 and a ticket more.  Heads of 256 in 8 and 4 bits have no tiles of 16."""
    native, need = pkg._native, {}
    cache = native.qcache(0x1000, 0x1000, 0x1000, 0x1000, 0, 0, 1 << 20, 1, 1, D, 1 << 20, 0, 0, 0, *bits, 1)
    args = native.qcache_attend_args(0x1000, 0x1000, 0, 16 * D, 16 * D, 16, 1, 1 << 20, 0, 0, 0.125, 0.0)
    try:
        native.tune("qcache_cluster", -1)
        for columns in (8, 16):
            native.tune("qcache_columns", columns)
            need[columns] = native.lib.b2kv_qcache_attend_workspace_bytes(cache, args)
    finally:
        native.tune("qcache_columns", 0)
        native.tune("qcache_cluster", 0)
    assert (need[16] != need[8]) == wide and need[8] > 0


# ---- the decoder ----

def decoder(pkg, ctx, batch_size=2, context_size=32, kv_bits=(8, 4), ragged=True):
    """(model module, state) of a decoder of zeros with one head of 64 and two layers."""
    from llm_experiments_b200 import model

    cfg = model.DecoderConfig(vocab_size=64, context_size=context_size, embedding_dim=64, n_heads=1, n_layers=2)
    z = lambda *shape: np.zeros(shape, dtype=np.float32)  # noqa: E731
    layer = dict(ln1_gamma=z(64), ln1_beta=z(64), wq=z(64, 64), wk=z(64, 64), wv=z(64, 64), wo=z(64, 64), ln2_gamma=z(64), ln2_beta=z(64),
                 w1=z(64, 256), b1=z(256), w2=z(256, 64), b2=z(64))
    weights = model.weights_from_numpy(ctx, cfg, dict(embedding=z(64, 64), pos_encoding=model.positional_encoding(context_size, 64), layers=[layer, layer],
                                                      lnf_gamma=z(64), lnf_beta=z(64), out_proj=z(64, 64)))
    return model, model.decoder_state_create(ctx, cfg, weights, batch_size=batch_size, kv_bits=kv_bits, ragged=ragged)


def folder_config():
    return dict(architecture="GPTDecoder", vocab_size=64, context_size=32, embedding_dim=64, n_heads=1, n_layers=1)


def folder_weights():
    z = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)  # noqa: E731
    layer = dict(ln1_gamma=z(64), ln1_beta=z(64), wq=z(64, 64), wk=z(64, 64), wv=z(64, 64), wo=z(64, 64), ln2_gamma=z(64), ln2_beta=z(64),
                 w1=z(64, 256), b1=z(256), w2=z(256, 64), b2=z(64))
    return dict(embedding=z(64, 64), out_proj=z(64, 64), lnf_gamma=z(64), lnf_beta=z(64), **{f"layers.0.{k}": t for k, t in layer.items()})


@pytest.mark.parametrize("bits", [None, [8, 4], [4, 4]])
def test_kv_bits_of_a_model_folder(pkg, ctx, tmp_path, bits):
    """``config.json`` and ``model.safetensors`` through the registry: caches of these bits, or bfloat16 ones without the entry."""
    import json

    from llm_experiments_b200 import checkpoint

    (tmp_path / "config.json").write_text(json.dumps(folder_config() if bits is None else dict(folder_config(), kv_bits=bits)))
    checkpoint.write_safetensors(tmp_path / "model.safetensors", folder_weights())
    dec = pkg.gpu.load_model(ctx, tmp_path)
    (cache,) = dec.state.caches
    if bits is None:
        assert isinstance(cache, pkg.gpu.KVCache) and dec.state.kv_bits is None
    else:
        assert isinstance(cache, pkg.gpu.QuantKVCache) and [cache.k_bits, cache.v_bits] == bits and dec.state.kv_bits == tuple(bits)
        assert (cache.max_seq_len, cache.n_kv_heads, cache.head_dim) == (32, 1, 64)


@pytest.fixture()
def no_launches(pkg, monkeypatch):
    """Operators of a layer that only note that they were called."""
    from llm_experiments_b200 import decode_layer

    called = []
    for name in ("layernorm", "matmul", "flash_attention"):
        monkeypatch.setattr(decode_layer, name, lambda *a, _name=name, **kw: called.append(_name))
    return called


def test_a_prompt_that_is_refused_leaves_the_caches_as_they_were(pkg, ctx, no_launches):
    model, state = decoder(pkg, ctx)
    from llm_experiments_b200 import decode_layer
    for cache in state.caches:
        pkg.gpu.quant_cache_set_lengths(cache, [7, 20])

    def refused(text, batch, seq_len, width=64, dtype=torch.bfloat16):
        x = two(pkg, batch * seq_len, width, dtype)
        scratch = decode_layer.prompt_layer_scratch(ctx, batch * seq_len, width)
        with pytest.raises(ValueError, match=text):
            decode_layer.prompt_layer_step(ctx, state.caches[0], x, state.weights.layers[0], scratch, x, batch, seq_len)
        assert no_launches == []
        assert all(c.current_len == 20 and c.seq_lens.tolist() == [7, 20] for c in state.caches)

    refused("Cache is full: seq_len=33", 2, 33)
    refused("dimensions", 3, 10)
    refused("dimensions", 2, 10, width=128)
    refused("dtype", 2, 10, dtype=torch.float32)
    refused("seq_len", 2, 0)


def test_launches_of_a_step_over_quantised_caches(pkg, ctx, monkeypatch):
    """Counted where the operators of a layer are called: each is one kernel, and the write with lengths on the device a second one."""
    from llm_experiments_b200 import decode_layer

    model, state = decoder(pkg, ctx)
    called = []
    for name in ("layernorm", "matmul", "quant_cache_update", "attention_with_quant_cache"):
        monkeypatch.setattr(decode_layer, name, lambda *a, _name=name, **kw: called.append(_name))
    decode_layer.decoder_layer_step(ctx, state.caches[0], state.x, state.weights.layers[0], state.scratch, state.y)
    per_layer = len(called) + called.count("quant_cache_update")
    assert per_layer == 11 and model.launches_per_decode_step(state.cfg, state.kv_bits) == 1 + per_layer * 2 + 3
    assert model.launches_per_decode_step(state.cfg) == 1 + 8 * 2 + 3


def test_a_step_without_room_for_the_new_rows_is_refused(pkg, ctx, no_launches):
    """Scratch made for bfloat16 caches."""
    from llm_experiments_b200 import decode_layer

    model, state = decoder(pkg, ctx)
    plain = decode_layer.decoder_layer_scratch(ctx, 2, 64)
    with pytest.raises(ValueError, match="quantised=True"):
        decode_layer.decoder_layer_step(ctx, state.caches[0], state.x, state.weights.layers[0], plain, state.y)
    assert no_launches == [] and state.caches[0].current_len == 0


@pytest.mark.parametrize("bits", [8, "84", (8.5, 4), ("8", "4"), (None, 4)])
def test_kv_bits_that_are_no_pair_of_numbers(pkg, ctx, bits):
    from llm_experiments_b200 import registry

    with pytest.raises(ValueError, match="kv_bits"):
        decoder(pkg, ctx, kv_bits=bits)
    with pytest.raises(ValueError, match="kv_bits"):
        registry.build_model(ctx, dict(folder_config(), kv_bits=bits), folder_weights())
