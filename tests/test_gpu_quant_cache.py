"""Quantised key / value cache on the GPU against float64: what is held (bit for bit), what is read back, and attention over it - types,
bits, head sizes, layouts, lengths about the tiles' edges, masks that leave rows empty, values that do not belong into a mean."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from tests.kv_util import make_ctx

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16
BITS = [(4, 4), (8, 4), (8, 8)]


@pytest.fixture(scope="module")
def ctx(pkg):
    return make_ctx(pkg)


def two(pkg, t):
    return pkg.gpu.GPUBuffer2D(buffer=t, shape=tuple(t.shape), size=t.numel())


def one(pkg, t):
    return pkg.gpu.GPUBuffer1D(buffer=t, shape=tuple(t.shape), size=t.numel())


def np64(t):
    return t.double().cpu().numpy()


def rnd(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def make(pkg, ctx, B, T, G, D, dtype=BF, bits=(4, 4), block=0, layers=1, seed=0, spare=0):
    """A cache with lengths of its own; paged: blocks in a drawn order, `spare` of the pool not in the table."""
    need = B * -(-T // block) if block else 0
    cache = pkg.gpu.quant_cache_create(ctx, pkg.gpu.QuantKVCacheConfig(
        batch_size=B, max_seq_len=T, n_layers=layers, n_kv_heads=G, head_dim=D, dtype=dtype, k_bits=bits[0], v_bits=bits[1], ragged=True,
        block_size=block, n_blocks=need + spare if block else 0))
    if block:
        order = torch.randperm(need + spare, generator=torch.Generator().manual_seed(seed))[:need]
        cache.block_table.copy_(order.to(torch.int32).view(B, -1))
    return cache


def update(pkg, ctx, cache, k, v, **kw):
    pkg.gpu.batch_begin(ctx)
    pkg.gpu.quant_cache_update(ctx, cache, kw.pop("layer", 0), two(pkg, k), two(pkg, v), **kw)
    pkg.gpu.batch_commit(ctx)


def gather(pkg, ctx, cache, which, **kw):
    pkg.gpu.batch_begin(ctx)
    out = pkg.gpu.quant_cache_gather(ctx, cache, kw.pop("layer", 0), which, **kw)
    pkg.gpu.batch_commit(ctx)
    return out


def attend(pkg, ctx, cache, q, **kw):
    out = torch.full_like(q, float("nan"))
    pkg.gpu.batch_begin(ctx)
    pkg.gpu.attention_with_quant_cache(ctx, cache, kw.pop("layer", 0), two(pkg, q), two(pkg, out), **kw)
    pkg.gpu.batch_commit(ctx)
    return out


def filled(pkg, ctx, lens, T, G, D, dtype=BF, bits=(4, 4), block=0, seed=1, k_scale=1.0, v_scale=1.0):
    """(cache of these lengths, what it holds in float64 [B, T, G, D] of keys and values); rows behind the lengths are written too."""
    B = len(lens)
    cache = make(pkg, ctx, B, T, G, D, dtype, bits, block, seed=seed)
    k, v = rnd((B * T, G * D), dtype, seed, k_scale), rnd((B * T, G * D), dtype, seed + 1, v_scale)
    update(pkg, ctx, cache, k, v, tokens=T)
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    return cache, [qo.held(np64(x).reshape(B, T, G, D), b) for x, b in zip((k, v), bits)]


def check(got, q, held, lens, m, scale=None, softcap=0.0, window=0, slopes=None):
    """got and q [B * m, H * D] tensors."""
    K, V = held
    B, D = len(lens), K.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    dtype = "bf16" if got.dtype == BF else "f32"
    got, q = np64(got).reshape(B, m, -1, D), np64(q).reshape(B, m, -1, D)
    for b, n in enumerate(lens):
        out, mean, size = qo.attention(q[b], K[b, :n], V[b, :n], scale, softcap, window, slopes)
        # biases up to slope * n and the cap are rounded to fp32 like the scores
        extra = 2.0 ** -22 * (softcap + (np.max(slopes) * n if slopes is not None else 0.0))
        tol = qo.tolerance(out, mean, size, n, dtype, extra, np.abs(V[b, :n]).max(initial=0.0))
        bad = ~(np.abs(got[b] - out) <= tol)
        assert not bad.any(), (b, n, np.argwhere(bad)[:4].tolist(), got[b][bad][:4], out[bad][:4], tol[bad][:4])


# ---------------------------------------------------------------------------------------------------------------------
# into the cache and back
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype,block,n", [(BF, 0, 1), (BF, 16, 37), (F32, 0, 19), (F32, 5, 1)])
def test_rows_are_held_and_read_back_bit_for_bit(pkg, ctx, D, bits, dtype, block, n):
    B, T, G = 3, 61, 2
    lens = [0, 7, T - n]
    cache = make(pkg, ctx, B, T, G, D, dtype, bits, block, spare=3)
    for lay in cache.layers:  # what must be left alone
        for b in (lay.k_codes, lay.v_codes, lay.k_scales, lay.v_scales):
            b.buffer.view(torch.uint8).fill_(0x5A)
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    before = [gather(pkg, ctx, cache, w, pending=T).clone() for w in "kv"]
    rows = []
    for s in (3, 4):
        x = rnd((B * n, G * D), dtype, s) * torch.exp2(torch.randint(-60, 60, (B * n, G * D // 32), generator=torch.Generator().manual_seed(s)).cuda()
                                                       ).repeat_interleave(32, dim=1).to(dtype)
        x[0, :32] = 0                                         # a group of zeros
        x[0, 31] = -0.0
        rows.append(x.contiguous())
    update(pkg, ctx, cache, *rows, tokens=n)
    assert cache.seq_lens.tolist() == [x + n for x in lens] and cache.current_len == T
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    for which, x, b, old in zip("kv", rows, bits, before):
        got = gather(pkg, ctx, cache, which, pending=T)       # (pending: beyond the lengths, to see the rows behind too)
        want = qo.held(np64(x).reshape(B, n, G, D), b)
        for i, s in enumerate(lens):
            np.testing.assert_array_equal(np64(got[i, s:s + n]), np64(torch.from_numpy(want[i]).to(dtype)))  # (16 bits: one rounding)
            assert torch.equal(got[i, :s].view(torch.uint8), old[i, :s].view(torch.uint8)) and torch.equal(got[i, s + n:].view(torch.uint8), old[i, s + n:].view(torch.uint8))
        tail = gather(pkg, ctx, cache, which, length=n + 2, last=True, pending=n)
        for i, s in enumerate(lens):
            np.testing.assert_array_equal(np64(tail[i, 2:]), np64(got[i, s:s + n]))
            assert s or not tail[i, :2].any()
        short = gather(pkg, ctx, cache, which)
        for i, s in enumerate(lens):
            assert torch.equal(short[i, :s].view(torch.uint8), old[i, :s].view(torch.uint8)) and not short[i, s:].view(torch.uint8).any()


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quotients_on_and_next_to_borders(pkg, ctx, bits, dtype):
    """Scales with every mantissa, and in each group quotients that are a border n + 1/2, or the next number of the type either side."""
    G, D = 1, 128
    rows, tops = 512, [7 if b == 4 else 127 for b in bits]
    gen = torch.Generator().manual_seed(5)
    cache = make(pkg, ctx, 1, rows, G, D, dtype, bits)
    ins = []
    for top in tops:
        scale = torch.exp2(torch.randint(-20, 20, (rows, 4), generator=gen).float()) * (1 + torch.randint(0, 128, (rows, 4), generator=gen) / 128)
        border = torch.randint(-top, top, (rows, 4, 32), generator=gen) + 0.5
        x = (border * scale[..., None]).to(dtype)
        up = torch.randint(-1, 2, x.shape, generator=gen)
        x = torch.where(up == 0, x, torch.nextafter(x, torch.where(up > 0, torch.inf, -torch.inf).to(dtype)))
        x[..., 0] = (scale * top).to(dtype)                   # (which makes the scale, or one next to it)
        ins.append(x.reshape(rows, D).cuda())
    update(pkg, ctx, cache, *ins, tokens=rows)
    for which, x, b in zip("kv", ins, bits):
        want = torch.from_numpy(qo.held(np64(x).reshape(1, rows, G, D), b)).to(dtype)
        assert torch.equal(gather(pkg, ctx, cache, which).cpu(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_groups_that_are_not_finite_read_back_as_nan(pkg, ctx, dtype):
    cache = make(pkg, ctx, 1, 6, 1, 64, dtype, (8, 4))
    x = rnd((6, 64), dtype, 1)
    x[1, 3], x[2, 40], x[3, 0], x[4, :] = float("inf"), float("nan"), -float("inf"), torch.finfo(dtype).max
    update(pkg, ctx, cache, x, x, tokens=6)
    for which, bits in (("k", 8), ("v", 4)):
        np.testing.assert_array_equal(np64(gather(pkg, ctx, cache, which)), np64(torch.from_numpy(qo.held(np64(x).reshape(1, 6, 1, 64), bits)).to(dtype)))


def test_rows_of_a_wider_buffer(pkg, ctx):
    """Keys, values and queries as columns of one projection's output."""
    B, H, G, D = 5, 6, 2, 64
    cache = make(pkg, ctx, B, 20, G, D)
    y = rnd((B, (H + 2 * G) * D), BF, 7)
    cut = lambda a, n: pkg.gpu.GPUBuffer2D(buffer=y[:, a * D:(a + n) * D], shape=(B, n * D), size=B * n * D)  # noqa: E731
    wide = torch.full((B, (H + 1) * D), 3.0, dtype=BF, device="cuda")
    pkg.gpu.batch_begin(ctx)
    pkg.gpu.quant_cache_update(ctx, cache, 0, cut(H, G), cut(H + G, G))
    pkg.gpu.attention_with_quant_cache(ctx, cache, 0, cut(0, H), pkg.gpu.GPUBuffer2D(buffer=wide[:, :H * D], shape=(B, H * D), size=B * H * D))
    pkg.gpu.batch_commit(ctx)
    held = [qo.held(np64(y[:, a * D:(a + G) * D]).reshape(B, 1, G, D), 4) for a in (H, H + G)]
    check(wide[:, :H * D], y[:, :H * D], held, [1] * B, 1)
    assert (wide[:, H * D:] == 3.0).all()


def test_places_and_blocks_outside_are_skipped_and_reported(pkg, ctx):
    gpu = pkg.gpu
    cache = make(pkg, ctx, 2, 32, 1, 64, block=16)
    rows = [rnd((64, 64), BF, i) for i in (1, 2)]
    update(pkg, ctx, cache, *rows, tokens=32)
    gpu.quant_cache_set_lengths(cache, [30, 20])
    good = gather(pkg, ctx, cache, "v")
    q = rnd((2, 64), BF, 3)
    fine = attend(pkg, ctx, cache, q)
    cache.block_table[0, 1] = 99
    ctx.dev_status.zero_()
    out = attend(pkg, ctx, cache, q)
    assert int(ctx.dev_status.item()) == 1 and torch.equal(out[1], fine[1])
    back = gather(pkg, ctx, cache, "v")
    assert torch.equal(back[0, :16], good[0, :16]) and not back[0, 16:].any() and torch.equal(back[1], good[1])
    held = [qo.held(np64(x).reshape(2, 32, 1, 64), 4) for x in rows]
    # the tokens of the block that is not there are as if they were masked: a query at place 29 sees the first 16
    want, mean, size = qo.attention(np64(q[:1]).reshape(1, 1, 64), held[0][0, :16], held[1][0, :16], 0.125)
    assert (np.abs(np64(out[0]) - want[0, 0]) <= qo.tolerance(want, mean, size, 16, "bf16")[0, 0]).all()
    ctx.dev_status.zero_()
    cache.seq_lens.copy_(torch.tensor([32, 20], dtype=torch.int32))  # the host's idea (30) is out of date: the device's place is full
    update(pkg, ctx, cache, q, q, advance=False)
    assert int(ctx.dev_status.item()) == 2
    ctx.dev_status.zero_()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------

LENS = [0, 1, 15, 16, 17, 31, 32, 33, 255, 256, 257, 300]


@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype,G,R", [(BF, 2, 1), (BF, 1, 12), (F32, 2, 3), (F32, 1, 9)])
def test_single_tokens(pkg, ctx, D, bits, dtype, G, R):
    cache, held = filled(pkg, ctx, LENS, 310, G, D, dtype, bits)
    q = rnd((len(LENS), G * R * D), dtype, 9, 1.5)
    check(attend(pkg, ctx, cache, q), q, held, LENS, 1)


@pytest.mark.parametrize("block", [0, 16, 24, 7])
@pytest.mark.parametrize("dtype,bits,D", [(BF, (4, 4), 128), (BF, (8, 8), 64), (F32, (8, 4), 96)])
@pytest.mark.parametrize("lens", [[2500], [1, 1023, 1024, 1025, 2049, 0, 4000]])
def test_long_rows_in_shares(pkg, ctx, block, dtype, bits, D, lens):
    cache, held = filled(pkg, ctx, lens, max(lens) + 3, 2, D, dtype, bits, block)
    q = rnd((len(lens), 4 * D), dtype, 9, 2.0)
    check(attend(pkg, ctx, cache, q), q, held, lens, 1)


@pytest.mark.parametrize("m", [2, 5, 8, 64])
@pytest.mark.parametrize("R", [1, 4, 7])
@pytest.mark.parametrize("dtype,window", [(BF, 0), (BF, 6), (F32, 40)])
def test_several_new_tokens(pkg, ctx, m, R, dtype, window):
    lens = [0, 1, m - 1, m, 33, 70, 257]
    cache, held = filled(pkg, ctx, lens, 300, 2, 64, dtype)
    q = rnd((len(lens) * m, 2 * R * 64), dtype, 9, 1.5)
    check(attend(pkg, ctx, cache, q, tokens=m, window=window), q, held, lens, m, window=window)


@pytest.mark.parametrize("window", [1, 16, 33, 1000, 5000])
@pytest.mark.parametrize("dtype,bits", [(BF, (4, 4)), (F32, (8, 8))])
def test_windows(pkg, ctx, window, dtype, bits):
    lens = [1, 16, 17, 48, 999, 1001, 2600]
    cache, held = filled(pkg, ctx, lens, 2600, 1, 64, dtype, bits, 16)
    q = rnd((len(lens), 3 * 64), dtype, 9, 1.5)
    check(attend(pkg, ctx, cache, q, window=window), q, held, lens, 1, window=window)


@pytest.fixture()
def tune(pkg):
    knobs = {}

    def set_knob(name, value):
        knobs[name] = 0
        pkg._native.tune(name, value)

    yield set_knob
    for name in knobs:
        pkg._native.tune(name, 0)


@pytest.mark.parametrize("cluster", [1, 2, 4, 8, -1])
@pytest.mark.parametrize("dtype,D,bits,block,m,R,window", [(BF, 128, (4, 4), 0, 1, 4, 0), (BF, 64, (8, 8), 16, 3, 5, 100), (F32, 96, (8, 4), 24, 2, 3, 0),
                                                           (BF, 256, (8, 4), 0, 1, 1, 0), (F32, 32, (4, 4), 64, 1, 9, 0)])
def test_every_way_to_cut(pkg, ctx, tune, cluster, dtype, D, bits, block, m, R, window):
    """CTAs in clusters and runs of tiles over many sequences: pairs cut once, several times and not at all, runs that begin anywhere."""
    tune("qcache_cluster", cluster)
    lens = [700, 0, 1, 33, 64, 1999, 5, 310, 96, 2, 0, 1024, 31, 32, 500]
    cache, held = filled(pkg, ctx, lens, 2000, 3, D, dtype, bits, block)
    q = rnd((len(lens) * m, 3 * R * D), dtype, 9, 1.5)
    check(attend(pkg, ctx, cache, q, tokens=m, window=window), q, held, lens, m, window=window)


@pytest.mark.parametrize("cluster", [3, 5, 6, 7])
@pytest.mark.parametrize("dtype,D,bits,m,R,columns", [(BF, 128, (8, 4), 1, 3, 0), (BF, 32, (4, 4), 5, 3, 0), (BF, 256, (8, 8), 4, 4, 16), (F32, 256, (4, 4), 1, 4, 0),
                                                      (F32, 32, (8, 8), 1, 1, 0), (BF, 96, (4, 4), 2, 5, 16), (F32, 64, (8, 4), 3, 2, 0)])
def test_clusters_that_do_not_divide_the_elements(pkg, ctx, tune, cluster, dtype, D, bits, m, R, columns):
    tune("qcache_cluster", cluster)
    tune("qcache_columns", columns)
    lens = [700, 0, 1, 33, 64, 1999, 5, 310]
    cache, held = filled(pkg, ctx, lens, 2000, 3, D, dtype, bits)
    q = rnd((len(lens) * m, 3 * R * D), dtype, 9, 1.5)
    check(attend(pkg, ctx, cache, q, tokens=m), q, held, lens, m)


@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("cluster,m,R", [(-1, 1, 16), (2, 5, 5), (1, 1, 3)])
def test_sixteen_columns(pkg, ctx, tune, D, bits, cluster, m, R):
    tune("qcache_columns", 16)
    tune("qcache_cluster", cluster)
    lens = [700, 0, 33, 64, 311, 5]
    cache, held = filled(pkg, ctx, lens, 700, 2, D, BF, bits, 16)
    q = rnd((len(lens) * m, 2 * R * D), BF, 9, 1.5)
    check(attend(pkg, ctx, cache, q, tokens=m), q, held, lens, m)


@pytest.mark.parametrize("lens", [[5000], [7001, 3], [0, 1], [16]])
@pytest.mark.parametrize("dtype,bits,D", [(BF, (4, 4), 128), (F32, (8, 4), 64)])
def test_few_pairs_in_even_pieces(pkg, ctx, tune, lens, dtype, bits, D):
    """Fewer pieces than CTAs that are there."""
    tune("qcache_cluster", -1)
    cache, held = filled(pkg, ctx, lens, max(lens) + 1, 1, D, dtype, bits)
    q = rnd((len(lens), 3 * D), dtype, 9, 2.0)
    check(attend(pkg, ctx, cache, q), q, held, lens, 1)


def test_more_sequences_than_threads(pkg, ctx, tune):
    """Runs over 500 sequences: every thread of a CTA adds up several."""
    lens = [(7 * i) % 61 for i in range(500)]
    for cluster in (-1, 1):
        tune("qcache_cluster", cluster)
        cache, held = filled(pkg, ctx, lens, 61, 1, 64)
        q = rnd((len(lens), 2 * 64), BF, 9, 1.5)
        check(attend(pkg, ctx, cache, q), q, held, lens, 1)


def test_a_window_longer_than_any_number(pkg, ctx):
    cache, held = filled(pkg, ctx, [90, 300], 300, 1, 64)
    q = rnd((2, 128), BF, 9)
    assert torch.equal(attend(pkg, ctx, cache, q, window=2 ** 31 - 1), attend(pkg, ctx, cache, q))


@pytest.mark.parametrize("softcap,biased", [(30.0, False), (0.5, True), (0.0, True)])
@pytest.mark.parametrize("dtype,m", [(BF, 1), (F32, 1), (BF, 3)])
def test_capped_and_biased_scores(pkg, ctx, softcap, biased, dtype, m):
    lens, H = [1, 40, 1500], 12
    cache, held = filled(pkg, ctx, lens, 1500, 4, 128, dtype, (8, 4), k_scale=3.0)
    q = rnd((3 * m, H * 128), dtype, 9, 3.0)
    slopes = torch.exp2(-8.0 * torch.arange(1, H + 1) / H).cuda() if biased else None
    got = attend(pkg, ctx, cache, q, tokens=m, softcap=softcap, slopes=None if slopes is None else one(pkg, slopes), scale=0.25)
    check(got, q, held, lens, m, 0.25, softcap, slopes=None if slopes is None else np64(slopes))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sizes_far_from_one(pkg, ctx, dtype):
    """Queries and keys of 2^60 and 2^-60, values of 2^-100 .. 2^100, values that differ by 2^12 between tokens and between groups."""
    lens, T, D = [70, 300], 300, 128
    B, G = 2, 2
    cache = make(pkg, ctx, B, T, G, D, dtype)
    k, v = rnd((B * T, G * D), dtype, 1, 2.0 ** -60), rnd((B * T, G * D), dtype, 2, 1.0)
    v *= torch.exp2(torch.randint(-6, 7, (B * T, 1), generator=torch.Generator().manual_seed(3)).float()).cuda().to(dtype)
    v[:, :32] *= 2.0 ** -12
    for by in (2.0 ** -100, 1.0, 2.0 ** 100):
        rows = (v.float() * by).to(dtype)
        pkg.gpu.quant_cache_reset(cache)
        update(pkg, ctx, cache, k, rows, tokens=T)
        pkg.gpu.quant_cache_set_lengths(cache, lens)
        held = [qo.held(np64(x).reshape(B, T, G, D), 4) for x in (k, rows)]
        q = rnd((B, 4 * D), dtype, 9, 2.0 ** 60)
        check(attend(pkg, ctx, cache, q), q, held, lens, 1)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scores_that_grow_along_the_sequence(pkg, ctx, dtype):
    """Every stage's scores outgrow the last one's by far, and one token outweighs all."""
    n, D = 700, 64
    cache = make(pkg, ctx, 1, n, 1, D, dtype, (8, 8))
    k = torch.ones((n, D), device="cuda") * torch.arange(n, device="cuda")[:, None] * 0.25
    k[300] = 400.0
    k, v = k.to(dtype), rnd((n, D), dtype, 2)
    update(pkg, ctx, cache, k, v, tokens=n)
    held = [qo.held(np64(x).reshape(1, n, 1, D), 8) for x in (k, v)]
    q = torch.ones((1, 2 * D), device="cuda", dtype=dtype)
    q[0, D:] = -1.0
    for w in (0, 350):
        check(attend(pkg, ctx, cache, q, window=w), q, held, [n], 1, window=w)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 64)])
def test_nan_stays_where_it_is_not_seen(pkg, ctx, dtype, D):
    """Tokens behind the end, outside the window or behind a drafted token's place hold NaN; so do blocks that no table names."""
    lens, T, m = [5, 40, 100], 128, 3
    cache, held = filled(pkg, ctx, lens, T, 1, D, dtype, block=16)
    bad = torch.full((3 * T, D), float("nan"), dtype=dtype, device="cuda")
    q = rnd((3 * m, 2 * D), dtype, 9)
    fine = attend(pkg, ctx, cache, q, tokens=m, window=20)
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    update(pkg, ctx, cache, bad[:3 * 28], bad[:3 * 28], tokens=28, advance=False)     # behind the ends
    assert torch.equal(attend(pkg, ctx, cache, q, tokens=m, window=20), fine)
    pkg.gpu.quant_cache_set_lengths(cache, [0, 0, 0])
    update(pkg, ctx, cache, bad[:3 * 78], bad[:3 * 78], tokens=78, advance=False)     # the third sees 78 .. 99 alone
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    got = attend(pkg, ctx, cache, q, tokens=m, window=20)
    assert torch.equal(got[2 * m:], fine[2 * m:]) and torch.isnan(got[:2 * m]).all()
    pkg.gpu.quant_cache_set_lengths(cache, [2, 10, 97])                                # the newest tokens: the first draft does not see them
    cache2, held2 = filled(pkg, ctx, lens, T, 1, D, dtype, block=16)
    pkg.gpu.quant_cache_set_lengths(cache2, [x - 2 for x in lens])
    update(pkg, ctx, cache2, bad[:6], bad[:6], tokens=2)
    got = attend(pkg, ctx, cache2, q, tokens=m).view(3, m, -1)
    want = attend(pkg, ctx, filled(pkg, ctx, lens, T, 1, D, dtype, block=16)[0], q, tokens=m).view(3, m, -1)
    assert torch.isnan(got[:, 1:]).all()
    tol = 2.0 ** -7 if dtype == BF else 2.0 ** -18  # the same sums in another order at most
    assert ((got[:, 0] - want[:, 0]).abs() <= tol * (want[:, 0].abs() + 1)).all()


def test_a_nan_value_group_spoils_its_elements_alone(pkg, ctx):
    cache = make(pkg, ctx, 1, 50, 1, 128)
    k, v = rnd((50, 128), BF, 1), rnd((50, 128), BF, 2)
    v[20, 70] = float("nan")
    update(pkg, ctx, cache, k, v, tokens=50)
    got = attend(pkg, ctx, cache, rnd((1, 256), BF, 3)).view(2, 128)
    assert torch.isnan(got[:, 64:96]).all() and torch.isfinite(got[:, :64]).all() and torch.isfinite(got[:, 96:]).all()


def test_a_query_that_is_not_finite_spoils_its_head_alone(pkg, ctx):
    cache, held = filled(pkg, ctx, [90], 90, 1, 64)
    q = rnd((1, 4 * 64), BF, 3)
    fine = attend(pkg, ctx, cache, q)
    q[0, 70] = float("inf")
    q[0, 130] = float("nan")
    got = attend(pkg, ctx, cache, q)
    assert torch.equal(got[0, :64], fine[0, :64]) and torch.equal(got[0, 192:], fine[0, 192:]) and torch.isnan(got[0, 64:192]).all()


def test_the_same_call_gives_the_same_bits(pkg, ctx):
    cache, _ = filled(pkg, ctx, [3000, 100, 1700], 3000, 2, 128, block=16)
    q = rnd((3, 8 * 128), BF, 3)
    first = attend(pkg, ctx, cache, q)
    for _ in range(3):
        assert torch.equal(attend(pkg, ctx, cache, q), first)


@pytest.mark.parametrize("dtype,m,R,lens", [(BF, 1, 4, [40, 0, 300]), (BF, 3, 7, [2500, 33, 900]), (F32, 2, 3, [700, 5, 64])])
@pytest.mark.parametrize("cluster", [1, 4, -1])
def test_outputs_in_the_queries_place(pkg, ctx, tune, dtype, m, R, lens, cluster):
    """Several tiles of columns and several CTAs to a pair, which write where others read their queries."""
    tune("qcache_cluster", cluster)
    cache, _ = filled(pkg, ctx, lens, max(lens), 2, 128, dtype)
    q = rnd((len(lens) * m, 2 * R * 128), dtype, 5, 1.5)
    want, both = attend(pkg, ctx, cache, q, tokens=m), two(pkg, q.clone())
    pkg.gpu.batch_begin(ctx)
    pkg.gpu.attention_with_quant_cache(ctx, cache, 0, both, both, tokens=m)
    pkg.gpu.batch_commit(ctx)
    assert torch.equal(both.buffer, want)


def test_buffers_that_lie_elsewhere_between_calls(pkg, ctx):
    """A layer's tensors may be given other memory; the next call goes there."""
    cache, _ = filled(pkg, ctx, [40, 7], 64, 2, 64)
    q = rnd((2, 4 * 64), BF, 5)
    want, layer = attend(pkg, ctx, cache, q), cache.layers[0]
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        t = getattr(layer, name).buffer
        moved = t.clone()
        old = t.detach().view_as(t)  # (keeps the old memory, which holds nothing of use any more)
        t.set_(moved)
        old.zero_()
    assert torch.equal(attend(pkg, ctx, cache, q), want)


def test_rows_whose_offsets_pass_32_bits(pkg, ctx):
    """The last sequence's rows lie beyond 4 GB of codes."""
    B, G, D, T = 3, 8, 128, 3_000_000
    cache = make(pkg, ctx, B, T, G, D)
    assert cache.layers[0].k_codes.buffer.numel() > 2 ** 32
    n = 100
    k, v = rnd((B * n, G * D), BF, 1), rnd((B * n, G * D), BF, 2)
    pkg.gpu.quant_cache_set_lengths(cache, [T - n, 0, T - n])
    update(pkg, ctx, cache, k, v, tokens=n)
    held = [qo.held(np64(x).reshape(B, n, G, D), 4) for x in (k, v)]
    for which, want in zip("kv", held):
        np.testing.assert_array_equal(np64(gather(pkg, ctx, cache, which, length=n, last=True)), np64(torch.from_numpy(want).to(BF)))
    q = rnd((B, G * D), BF, 3)
    check(attend(pkg, ctx, cache, q, window=n), q, held, [n] * B, 1)


# ---------------------------------------------------------------------------------------------------------------------
# used together
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,block", [(BF, 0), (F32, 16)])
def test_a_prompt_and_a_decoding_loop_over_two_layers(pkg, ctx, dtype, block):
    """Prompt rows into both layers, then tokens one and two at a time: every layer is written before it attends, the last one advances."""
    gpu, B, H, D, N = pkg.gpu, 3, 4, 64, 45
    cache = make(pkg, ctx, B, 80, H, D, dtype, (8, 4), block, layers=2)
    held = []
    for layer in range(2):
        q, k, v = (rnd((B * N, H * D), dtype, 10 * layer + i) for i in range(3))
        out = torch.empty_like(q)
        gpu.batch_begin(ctx)
        gpu.flash_attention(ctx, two(pkg, q), two(pkg, k), two(pkg, v), two(pkg, out), None, None, B, N, H, D)
        gpu.quant_cache_update(ctx, cache, layer, two(pkg, k), two(pkg, v), tokens=N, advance=layer == 1)
        gpu.batch_commit(ctx)
        held.append([qo.held(np64(x).reshape(B, N, H, D), b) for x, b in ((k, 8), (v, 4))])
    n = N
    for step, m in enumerate((1, 2, 1)):
        outs = []
        gpu.batch_begin(ctx)
        for layer in range(2):
            q, k, v = (rnd((B * m, H * D), dtype, 100 * step + 10 * layer + i + 50) for i in range(3))
            out = torch.empty_like(q)
            last = layer == 1
            gpu.quant_cache_update(ctx, cache, layer, two(pkg, k), two(pkg, v), tokens=m, advance=last)
            gpu.attention_with_quant_cache(ctx, cache, layer, two(pkg, q), two(pkg, out), tokens=m, pending=0 if last else m)
            outs.append((q, out))
            held[layer] = [np.concatenate([old, qo.held(np64(x).reshape(B, m, H, D), b)], axis=1) for old, x, b in zip(held[layer], (k, v), (8, 4))]
        gpu.batch_commit(ctx)
        n += m
        assert cache.current_len == n and cache.seq_lens.tolist() == [n] * B
        for layer, (q, out) in enumerate(outs):
            check(out, q, held[layer], [n] * B, m)


def test_shared_host_length(pkg, ctx):
    """A cache without lengths of its own, as the reference's."""
    gpu = pkg.gpu
    cache = gpu.quant_cache_create(ctx, gpu.QuantKVCacheConfig(batch_size=2, max_seq_len=50, n_layers=1, n_kv_heads=1, head_dim=64, k_bits=8, v_bits=8))
    k, v = rnd((2 * 33, 64), BF, 1), rnd((2 * 33, 64), BF, 2)
    update(pkg, ctx, cache, k, v, tokens=33)
    assert cache.current_len == 33
    q = rnd((2, 64), BF, 3)
    check(attend(pkg, ctx, cache, q), q, [qo.held(np64(x).reshape(2, 33, 1, 64), 8) for x in (k, v)], [33, 33], 1)


def test_replayed_from_two_graphs_at_once(pkg, ctx):
    """Steps captured from two caches, replayed on two streams side by side, lengths moving on the device: as the same steps one by one."""
    gpu, D, G, H, steps = pkg.gpu, 128, 2, 8, 5

    def state(seed):
        lens = [2100 + seed, 40]
        cache, _ = filled(pkg, ctx, lens, 2200, G, D, seed=seed)
        ins = [rnd((steps, 2, n * D), BF, seed + 20 + i) for i, n in enumerate((H, G, G))]
        feed = [torch.zeros_like(x[0]) for x in ins]
        return cache, ins, feed, torch.zeros((2, H * D), dtype=BF, device="cuda")

    def step(cache, feed, out):
        gpu.batch_begin(ctx)
        gpu.quant_cache_update(ctx, cache, 0, two(pkg, feed[1]), two(pkg, feed[2]))
        gpu.attention_with_quant_cache(ctx, cache, 0, two(pkg, feed[0]), two(pkg, out))
        gpu.batch_commit(ctx)

    want = []
    for seed in (1, 2):
        cache, ins, feed, out = state(seed)
        for i in range(steps):
            cache.current_len = 2199
            for f, x in zip(feed, ins):
                f.copy_(x[i])
            step(cache, feed, out)
            want.append(out.clone())
    graphs, states = [], [state(1), state(2)]
    for cache, ins, feed, out in states:
        keep = cache.seq_lens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.current_len = 2199
            step(cache, feed, out)
            cache.seq_lens.copy_(keep)
            cache.current_len = 2199
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(cache, feed, out)
            cache.seq_lens.copy_(keep)
        graphs.append((graph, side))
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for (graph, side), (cache, ins, feed, out), mine in zip(graphs, states, got):
            with torch.cuda.stream(side):
                for f, x in zip(feed, ins):
                    f.copy_(x[i])
                graph.replay()
                mine.append(out.clone())
    torch.cuda.synchronize()
    for a, b in zip(want, got[0] + got[1]):
        assert torch.equal(a, b)
