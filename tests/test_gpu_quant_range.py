"""Attention over a quantised cache at the ends of its inputs' ranges, against float64: values near the type's largest, groups and tokens whose
values lie far apart, large values that no weight or no query reaches, queries, keys and caps at the ends of the type."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from tests.test_gpu_quant_cache import BF, F32, attend, filled, make, np64, one, rnd, tune, update  # noqa: F401  (tune: a fixture)
from tests.kv_util import make_ctx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pkg):
    return make_ctx(pkg)


def holding(pkg, ctx, lens, T, k, v, D, dtype, bits):
    """(cache with these lengths and rows [B * T, G * D], what it holds)."""
    B, G = len(lens), k.shape[1] // D
    cache = make(pkg, ctx, B, T, G, D, dtype, bits)
    update(pkg, ctx, cache, k, v, tokens=T)
    pkg.gpu.quant_cache_set_lengths(cache, lens)
    return cache, [qo.held(np64(x).reshape(B, T, G, D), b) for x, b in zip((k, v), bits)]


def check(got, q, held, lens, m, scale=None, softcap=0.0, window=0, extra=0.0, ordinary=None):
    """ordinary [B, T]: the tokens that a group's reference goes by, where the others are known to be too large for it and too few to move it."""
    K, V = held
    B, D = len(lens), K.shape[-1]
    dtype = "bf16" if got.dtype == BF else "f32"
    got, q = np64(got).reshape(B, m, -1, D), np64(q).reshape(B, m, -1, D)
    for b, n in enumerate(lens):
        out, mean, size = qo.attention(q[b], K[b, :n], V[b, :n], D ** -0.5 if scale is None else scale, softcap, window)
        counted = V[b, :n] if ordinary is None else V[b, :n] * ordinary[b, :n, None, None]
        tol = qo.tolerance_seen(out, mean, size, n, dtype, qo.largest_seen(counted, m, out.shape[1], window), extra)
        bad = ~(np.abs(got[b] - out) <= tol)
        assert not bad.any(), (b, n, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[b][bad][:4], out[bad][:4], tol[bad][:4])


def times(v, exponents):
    return (v.float() * torch.exp2(exponents.float().to(v.device))).to(v.dtype)


# ---------------------------------------------------------------------------------------------------------------------
# values far apart
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,bits,columns", [(128, (4, 4), 0), (128, (8, 8), 16), (64, (8, 4), 0), (96, (4, 4), 0), (256, (8, 8), 0), (256, (4, 4), 16), (32, (4, 4), 0)])
@pytest.mark.parametrize("apart", [12, 20, 30, 90])
def test_groups_that_lie_far_apart(pkg, ctx, tune, dtype, D, bits, columns, apart):  # noqa: F811
    tune("qcache_columns", columns)
    lens, T, G, R = [70, 1, 300, 33], 300, 2, 3
    k, v = rnd((4 * T, G * D), dtype, 1), rnd((4 * T, G * D), dtype, 2)
    v = times(v, apart * ((torch.arange(G * D) // 32) % 3 - 1).repeat(4 * T, 1))
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, bits)
    q = rnd((4, G * R * D), dtype, 3, 1.5)
    check(attend(pkg, ctx, cache, q), q, held, lens, 1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,bits", [(128, (4, 4)), (64, (8, 8)), (96, (8, 4))])
@pytest.mark.parametrize("cluster", [1, -1])
@pytest.mark.parametrize("shape", ["any", "up", "down", "first", "last", "few", "two"])
def test_tokens_that_lie_far_apart(pkg, ctx, tune, dtype, D, bits, cluster, shape):  # noqa: F811
    """Values' magnitudes along a sequence: anywhere for each token and group, rising, falling, one at the front or the end, a few, two sizes by turns."""
    tune("qcache_cluster", cluster)
    lens, T = [700, 45, 3], 700
    B, t = len(lens), torch.arange(T)
    gen = torch.Generator().manual_seed(4)
    by_token = {"any": lambda: torch.randint(-40, 41, (B * T, D // 32), generator=gen).repeat_interleave(32, 1),
                "up": lambda: (t // 7 - 50).repeat(B)[:, None], "down": lambda: (50 - t // 7).repeat(B)[:, None],
                "first": lambda: torch.where(t == 0, 30, 0).repeat(B)[:, None], "last": lambda: torch.cat([torch.where(t == n - 1, 30, 0) for n in lens])[:, None],
                "few": lambda: torch.where(t % 97 == 5, 90, -20).repeat(B)[:, None], "two": lambda: (t % 2 * 25).repeat(B)[:, None]}[shape]()
    k, v = rnd((B * T, D), dtype, 1), times(rnd((B * T, D), dtype, 2), by_token.expand(B * T, -1) if by_token.shape[1] == 1 else by_token)
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, bits)
    q = rnd((B, 4 * D), dtype, 3, 1.5)
    check(attend(pkg, ctx, cache, q), q, held, lens, 1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("large", [20, 40, 100])
@pytest.mark.parametrize("away", [25.0, 80.0])
def test_large_values_of_tokens_with_next_to_no_weight(pkg, ctx, dtype, large, away):
    """Tokens whose scores lie `away` below all others': their weight is e^-25 (times 2^40 it counts again) or nothing that counts."""
    lens, T, D = [200, 40], 200, 64
    k, v = rnd((2 * T, D), dtype, 1, 0.3), rnd((2 * T, D), dtype, 2)
    off = torch.arange(2 * T, device="cuda") % 17 == 3
    k[:, 0] = torch.where(off, -away / 4.0, 0.0).to(dtype)        # times 32 and 64 ** -0.5
    v = times(v, torch.where(off, large, 0)[:, None].expand(-1, D))
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, (8, 8))
    q = rnd((2, 2 * D), dtype, 3)
    q.view(2, 2, D)[:, :, 0] = 32.0
    check(attend(pkg, ctx, cache, q), q, held, lens, 1, ordinary=~off.view(2, T).cpu().numpy())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("large", [40, 120])
@pytest.mark.parametrize("bits,window", [((4, 4), 0), ((8, 8), 0), ((8, 4), 25)])
def test_large_values_that_a_query_does_not_see(pkg, ctx, dtype, large, bits, window):
    """A later drafted token's values, or those before the window, are no part of an earlier query's mean, whatever their size."""
    lens, T, D, m = [20, 64, 300], 300, 128, 3
    k, v = rnd((3 * T, D), dtype, 1), rnd((3 * T, D), dtype, 2)
    big = torch.zeros((3, T), dtype=torch.int64)
    for b, n in enumerate(lens):
        big[b, n - 1] = large
        if window:
            big[b, :max(0, n - m + 1 - window)] = large - 3
    v = times(v, big.view(-1, 1).expand(-1, D))
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, bits)
    q = rnd((3 * m, 4 * D), dtype, 3, 1.5)
    check(attend(pkg, ctx, cache, q, tokens=m, window=window), q, held, lens, m, window=window)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cluster", [-1, 1])
def test_sequences_of_other_sizes_one_after_another(pkg, ctx, tune, dtype, cluster):  # noqa: F811
    """A CTA that goes through many sequences starts each with references of its own; some sequences are empty, some all zeros, some hold one NaN."""
    tune("qcache_cluster", cluster)
    lens, T, D = [(7 * i) % 61 for i in range(700)], 61, 64
    B, i = len(lens), torch.arange(len(lens))
    k, v = rnd((B * T, D), dtype, 1), rnd((B * T, D), dtype, 2)
    v = times(v, ((i * 37) % 161 - 80).repeat_interleave(T)[:, None].expand(-1, D))
    v.view(B, T, D)[5::50] = 0
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, (8, 4))
    q = rnd((B, 2 * D), dtype, 3, 1.5)
    fine = attend(pkg, ctx, cache, q)
    check(fine, q, held, lens, 1)
    v.view(B, T, D)[9::50, 0, 40] = float("nan")
    got = attend(pkg, ctx, holding(pkg, ctx, lens, T, k, v, D, dtype, (8, 4))[0], q).view(B, 2, D)
    struck = [b for b in range(9, B, 50) if lens[b] > 0]
    assert torch.isnan(got[struck][:, :, 32:]).all() and torch.equal(got[struck][:, :, :32], fine.view(B, 2, D)[struck][:, :, :32])
    others = [b for b in range(B) if b not in struck]
    assert torch.equal(got[others], fine.view(B, 2, D)[others])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_beside_values_far_apart(pkg, ctx, dtype):
    lens, T, D = [90], 90, 128
    k, v = rnd((T, D), dtype, 1), times(rnd((T, D), dtype, 2), torch.randint(-30, 31, (T, 4), generator=torch.Generator().manual_seed(5)).repeat_interleave(32, 1))
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, (8, 4))
    q = rnd((1, 2 * D), dtype, 3)
    fine = attend(pkg, ctx, cache, q).view(2, D)
    v[20, 70] = float("nan")
    got = attend(pkg, ctx, holding(pkg, ctx, lens, T, k, v, D, dtype, (8, 4))[0], q).view(2, D)
    assert torch.isnan(got[:, 64:96]).all()
    assert torch.equal(got[:, :64], fine[:, :64]) and torch.equal(got[:, 96:], fine[:, 96:])


@pytest.mark.parametrize("dtype,D,bits", [(BF, 128, (4, 4)), (F32, 64, (8, 8)), (BF, 256, (8, 4)), (F32, 96, (8, 4))])
@pytest.mark.parametrize("cluster", [1, 2, 8, -1])
@pytest.mark.parametrize("lens", [[20, 700], [9000]])
def test_values_near_the_largest_number(pkg, ctx, tune, dtype, D, bits, cluster, lens):  # noqa: F811
    """A mean of values lies among them, however large they are."""
    tune("qcache_cluster", cluster)
    B, T = len(lens), max(lens)
    k, v = rnd((B * T, D), dtype, 1, 0.2), rnd((B * T, D), dtype, 2)
    v = (torch.where(v < -1.5, -3.0e38, 3.0e38) * torch.rand(v.shape, generator=torch.Generator("cuda").manual_seed(3), device="cuda")).to(dtype)
    v[:, ::16] = 3.0e38
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, bits)
    q = rnd((B, 2 * D), dtype, 3)
    check(attend(pkg, ctx, cache, q), q, held, lens, 1)


# ---------------------------------------------------------------------------------------------------------------------
# queries and caps
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits,q_exp,k_exp,scale", [((4, 4), 119, -120, 1.0), ((8, 8), 117, -118, 1.0), ((4, 4), 124, -122, 0.18), ((8, 4), 124, -118, 2.0 ** -6),
                                                    ((4, 4), -112, 112, 0.18), ((8, 8), -115, 115, 0.18), ((4, 4), 100, 20, 2.0 ** -122), ((8, 8), -90, -25, 2.0 ** 113)])
@pytest.mark.parametrize("options", [{}, {"softcap": 20.0}, {"window": 40}])
def test_queries_at_the_ends_of_the_type(pkg, ctx, dtype, bits, q_exp, k_exp, scale, options):
    """Scores of ordinary size by the definition, from queries, keys and scales that are not."""
    lens, T, D = [70, 300, 1], 300, 32
    k, v = rnd((3 * T, D), dtype, 1), rnd((3 * T, D), dtype, 2)
    k = times(k, torch.full(k.shape, k_exp))
    cache, held = holding(pkg, ctx, lens, T, k, v, D, dtype, bits)
    q = rnd((3, 3 * D), dtype, 9)
    q[:, D:2 * D] = times(q[:, D:2 * D], torch.full((3, D), q_exp))
    q[:, 2 * D:] = times(q[:, 2 * D:], torch.full((3, D), q_exp - 1))
    q[:, :D] = 0.0                                                # (a head beside them whose scores are all 0)
    check(attend(pkg, ctx, cache, q, scale=scale, **options), q, held, lens, 1, scale, extra=2.0 ** -22 * options.get("softcap", 0.0), **options)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [1e-30, 1e-3, 1e10, 1e30, 1e37, 1e38, 2.4e38, float(torch.finfo(F32).max)])
@pytest.mark.parametrize("slopes", [False, True])
def test_every_cap_that_is_taken(pkg, ctx, dtype, cap, slopes):
    """A cap beyond all scores is none; one below them all leaves the tokens' mean (and the bias)."""
    lens, D = [1, 40, 500], 64
    cache, held = filled(pkg, ctx, lens, 500, 1, D, dtype, (8, 4))
    q = rnd((3, 2 * D), dtype, 9, 3.0)
    bias = torch.tensor([0.25, 0.01], device="cuda")
    got = attend(pkg, ctx, cache, q, softcap=cap, slopes=one(pkg, bias) if slopes else None)
    assert torch.isfinite(got).all()
    K, V = held
    got64, q64 = np64(got).reshape(3, 1, 2, D), np64(q).reshape(3, 1, 2, D)
    for b, n in enumerate(lens):
        out, mean, size = qo.attention(q64[b], K[b, :n], V[b, :n], D ** -0.5, cap, 0, np64(bias) if slopes else None)
        # scores (below 40) are rounded a few times on their way through the cap, the bias (up to n / 4) once; a cap near the type's largest number leaves
        # steps of 2^-149 in what tanh gets, 2^-23 of a score by a cap of 2^126 or less
        extra = 2.0 ** -22 * (min(cap, 40.0) + (0.25 * n if slopes else 0.0)) + 2.0 ** -22
        tol = qo.tolerance_seen(out, mean, size, n, "bf16" if dtype == BF else "f32", qo.largest_seen(V[b, :n], 1, 2), extra)
        assert (np.abs(got64[b] - out) <= tol).all(), (b, n, np.abs(got64[b] - out).max(), tol.min())
