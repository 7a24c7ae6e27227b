"""Attention over a quantised cache at the ends of its inputs' ranges, against float64."""
import pytest
import torch

from oracle import quant_cache_oracle as qo
from tests.kv_util import make_ctx
from tests.test_gpu_quant_cache import BF, F32, attend, check, make, np64, rnd, tune, update  # noqa: F401  (tune: a fixture)

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
