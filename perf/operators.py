"""Operators of a quantised key / value cache: what a pass through each reads and returns, in plain torch and through the framework.

A cached row of one key / value head is cut into groups of 32 elements.  A group is held as whole numbers of 4 or 8 bits and one
bfloat16 scale:

    scale = bf16(max |x| / L)        L = 7 for 4 bits, 127 for 8
    code  = x / scale to the nearest whole number (ties to even), within -L .. L; 0 where the scale is 0
    value = code * scale

A group that holds an infinity or a NaN has a NaN for its scale.  Kinds of case:

* ``attend``: attention of the last ``m`` tokens of every sequence over a cache in that form (``attention_with_quant_cache``).  Query i
  of a sequence with n tokens stands at place p = n - m + i and sees the tokens t <= p, with a window only those with p - t < window:
  score = cap(scale * q . k) - slope * (p - t), cap(x) = softcap * tanh(x / softcap).  A query that sees nothing gives zeros;
* ``write``: ``m`` new rows per sequence behind those it holds are quantised into the cache (``quant_cache_update``) and read back
  (``quant_cache_gather``), which is how a program that goes on over them in full width gets them;
* ``read``: a whole cache read back, zeros behind the end of each sequence.
"""
import importlib.util
import math
import pathlib
import sys

import numpy as np
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 32
own = False


def package():
    name = "llm_experiments_b200"  # the folder's name has a hyphen
    if name not in sys.modules:
        folder = ROOT / "llm-experiments_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py", submodule_search_locations=[str(folder)])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


_CTX = []


def context():
    if not _CTX:
        _CTX.append(package().gpu.context_create(0))
    return _CTX[0]


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------

def attend(name, B, H, G, D, lo, hi, dtype="bf16", kb=4, vb=4, block=0, m=1, window=0, softcap=0.0, slopes=False):
    """``B`` sequences of ``lo`` .. ``hi`` tokens, ``H`` query heads over ``G`` key / value heads of ``D`` elements."""
    return dict(name=name, kind="attend", B=B, H=H, G=G, D=D, lo=lo, hi=hi, dtype=dtype, kb=kb, vb=vb, block=block, m=m, window=window,
                softcap=softcap, slopes=slopes)


def write(name, B, G, D, m, lo, hi, dtype="bf16", kb=4, vb=4, block=0):
    """``m`` rows for each of ``B`` sequences that hold ``lo`` .. ``hi`` tokens."""
    return dict(name=name, kind="write", B=B, G=G, D=D, m=m, lo=lo, hi=hi, dtype=dtype, kb=kb, vb=vb, block=block)


def read(name, B, G, D, lo, hi, dtype="bf16", kb=4, vb=4, block=0):
    return dict(name=name, kind="read", B=B, G=G, D=D, lo=lo, hi=hi, dtype=dtype, kb=kb, vb=vb, block=block)


def listed():
    return [
        # The reference's own small model (4 heads of 64, fp32, batch of one) in the middle of a generation: nothing but latency.
        attend("attend_one_f32", B=1, H=4, G=4, D=64, lo=160, hi=160, dtype="f32"),
        # A handful of conversations with short histories, keys kept finer than values.
        attend("attend_few", B=8, H=32, G=8, D=128, lo=128, hi=1024, kb=8),
        # The benchmark's batch: 64 sequences of 512 .. 8192 tokens, every head with keys and values of its own.
        attend("attend_batch", B=64, H=32, G=32, D=128, lo=512, hi=8192),
        # A server with a block table: 16-token blocks anywhere in a pool, an odd number of sequences, smaller heads in 8 bits.
        attend("attend_paged", B=13, H=24, G=8, D=64, lo=301, hi=5003, kb=8, vb=8, block=16),
        # The benchmark's long contexts, grouped heads.
        attend("attend_long", B=4, H=64, G=8, D=128, lo=131072, hi=131072),
        # A design with capped scores, a distance bias and a sliding window.
        attend("attend_window", B=32, H=16, G=4, D=128, lo=700, hi=4000, kb=8, vb=8, window=1024, softcap=30.0, slopes=True),
        # Five drafted tokens per sequence looked over in one call.
        attend("attend_drafts", B=8, H=32, G=4, D=128, lo=1500, hi=2048, m=5),
        # Heads of 96 in the reference's storage type.
        attend("attend_f32", B=16, H=12, G=4, D=96, lo=1000, hi=4000, dtype="f32", kb=8),
        # One new token for each sequence of the benchmark's batch.
        write("write_token", B=64, G=32, D=128, m=1, lo=512, hi=8191),
        # The benchmark's prompts into an empty cache.
        write("write_prompt", B=8, G=32, D=128, m=4096, lo=0, hi=0),
        # Prompts in the reference's storage type, of a length that fills no block, behind a history.
        write("write_paged_f32", B=2, G=12, D=64, m=1000, lo=100, hi=300, dtype="f32", kb=8, vb=8, block=16),
        # A cache of odd lengths read back whole.
        read("read_ragged", B=13, G=8, D=128, lo=301, hi=5003, kb=8),
    ]


def spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "write", "write", "read"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    kb, vb = rng.choice([(4, 4), (4, 4), (8, 4), (8, 8)])
    common = dict(kind=kind, B=spread(rng, 1, 64), D=rng.choice([32, 64, 64, 96, 128, 128, 128, 256]), dtype=dtype, kb=kb, vb=vb,
                  block=rng.choice([0, 0, 0, 16, 64, 24]))
    if kind == "attend":
        G, hi = spread(rng, 1, 32), spread(rng, 1, 131072)
        c = dict(common, G=G, H=G * rng.choice([1, 1, 2, 3, 4, 6, 8, 16]), lo=0, hi=hi, m=rng.choice([1, 1, 1, rng.randint(2, 8)]),
                 window=rng.choice([0, 0, spread(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.25)
        while c["B"] * c["H"] * c["D"] * c["hi"] * c["m"] > 6e8:
            c["B" if c["B"] > 4 else "hi"] //= 2
        c["lo"] = rng.choice([c["hi"], c["hi"] // 16, c["hi"] // 16])
        return c
    c = dict(common, G=spread(rng, 1, 32), lo=0, hi=spread(rng, 1, 8192))
    if kind == "write":
        c["m"] = rng.choice([1, spread(rng, 1, 4096), spread(rng, 1, 4096)])
        while c["B"] * c["G"] * c["D"] * c["m"] > 1.3e8:
            c["m"] //= 2
        while c["B"] * c["G"] * c["D"] * c["hi"] > 1e9:
            c["hi"] //= 2
    else:
        while c["B"] * c["G"] * c["D"] * c["hi"] > 1.3e8:
            c["hi"] //= 2
    c["lo"] = rng.choice([c["hi"], c["hi"] // 16])
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + salt)


def lengths(c, seed):
    return np.random.default_rng(int(seed)).integers(c["lo"], c["hi"] + 1, size=c["B"]).tolist()


def capacity(c):
    return max(1, c["hi"] + (c["m"] if c["kind"] == "write" else 0))


def history(c, seed, which):
    """Rows ``[B * T, G * D]`` that the cache holds (those behind a sequence's length are never seen).  Some channels of keys are
    several times as large as the others, as they are in trained models."""
    gen = generator(seed, 11 if which == "k" else 12)
    rows = torch.empty((c["B"] * capacity(c), c["G"] * c["D"]), dtype=DTYPES[c["dtype"]], device="cuda").normal_(generator=gen)
    return rows.mul_(channels(c, seed).to(rows.dtype)) if which == "k" else rows


def channels(c, seed):
    gen = generator(seed, 13)
    big = torch.rand((c["G"] * c["D"],), generator=gen, device="cuda") < 0.03
    return torch.where(big, 4.0, 1.0)


def rows_in(c, seed):
    """The step's rows: queries, or new keys and values."""
    gen, dt = generator(seed, 14), DTYPES[c["dtype"]]
    if c["kind"] == "attend":
        return (torch.empty((c["B"] * c["m"], c["H"] * c["D"]), dtype=dt, device="cuda").normal_(generator=gen).mul_(1.5),)
    k, v = (torch.empty((c["B"] * c["m"], c["G"] * c["D"]), dtype=dt, device="cuda").normal_(generator=gen) for _ in range(2))
    return k.mul_(channels(c, seed).to(dt)), v


def slopes_of(c):
    """A distance bias that falls geometrically over the heads."""
    return torch.exp2(-8.0 * torch.arange(1, c["H"] + 1, dtype=torch.float64, device="cuda") / c["H"]).float() if c["slopes"] else None


def prepare(case, seed):
    c = case
    st = dict(c=c, lens=lengths(c, seed), slopes=slopes_of(c) if c["kind"] == "attend" else None)
    st["rows"] = rows_in(c, seed) if c["kind"] != "read" else ()
    held = c["hi"] > 0
    if not own:
        # codes [B, T, G, D] and scales [B, T, G, D / 32], as a plain program keeps them
        shape = (c["B"], capacity(c), c["G"], c["D"])
        for which, bits in (("k", c["kb"]), ("v", c["vb"])):
            if held:
                st[which] = tuple(t.view(*shape[:3], -1) for t in quantise(history(c, seed, which), bits, c["D"]))
            else:
                st[which] = (torch.zeros(shape, dtype=torch.int8, device="cuda"),
                             torch.zeros((*shape[:3], c["D"] // GROUP), dtype=torch.bfloat16, device="cuda"))
        return st
    gpu, ctx = package().gpu, context()
    T = capacity(c)
    cache = gpu.quant_cache_create(ctx, gpu.QuantKVCacheConfig(
        batch_size=c["B"], max_seq_len=T, n_layers=1, n_kv_heads=c["G"], head_dim=c["D"], dtype=DTYPES[c["dtype"]], k_bits=c["kb"],
        v_bits=c["vb"], ragged=True, block_size=c["block"]))
    if c["block"]:
        gen, n = generator(seed, 15), cache.block_table.numel()
        cache.block_table.copy_(torch.randperm(n, generator=gen, device="cuda").view(cache.block_table.shape))
    two = lambda t: gpu.GPUBuffer2D(buffer=t, shape=tuple(t.shape), size=t.numel())  # noqa: E731
    if held:
        gpu.batch_begin(ctx)
        gpu.quant_cache_update(ctx, cache, 0, two(history(c, seed, "k")), two(history(c, seed, "v")), tokens=T)
        gpu.batch_commit(ctx)
    gpu.quant_cache_set_lengths(cache, st["lens"])
    st.update(gpu=gpu, ctx=ctx, cache=cache, rows=[two(t) for t in st["rows"]])
    if c["kind"] == "attend":
        st["out"] = two(torch.empty_like(st["rows"][0].buffer))
        if c["slopes"]:
            st["slopes"] = gpu.GPUBuffer1D(buffer=st["slopes"], shape=(c["H"],), size=c["H"])
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------

def quantise(rows, bits, D):
    """(codes int8 [rows, heads, D], scales bf16 [rows, heads, D / 32]) of rows [rows, heads * D]."""
    top = 7 if bits == 4 else 127
    x = rows.float().view(rows.shape[0], -1, D // GROUP, GROUP)
    most = x.abs().amax(-1)
    # (by a tensor: torch divides by a number as a product with its reciprocal, which rounds twice)
    scales = torch.where(torch.isfinite(most), most / torch.full_like(most, top), torch.nan).to(torch.bfloat16)
    by = scales.float().unsqueeze(-1)
    codes = torch.where(by > 0, torch.round(x / by), 0.0).clamp(-top, top)
    return codes.view(*scales.shape[:2], D).to(torch.int8), scales


def values(codes, scales):
    """What codes stand for, fp32."""
    x = codes.float().view(*scales.shape, GROUP) * scales.float().unsqueeze(-1)
    return x.view(codes.shape)


def tokens_of(held, at):
    """Values [B, n, G, D] of the tokens at [B, n] (places before the first are those of the first)."""
    who = torch.arange(at.shape[0], device="cuda").unsqueeze(1)
    return values(*(t[who, at.clamp(min=0)] for t in held))


def plain_attend(st):
    c, (q,) = st["c"], st["rows"]
    B, m, H, G, D = c["B"], c["m"], c["H"], c["G"], c["D"]
    ends = torch.tensor(st["lens"], device="cuda").unsqueeze(1)
    span = max(1, max(visible(c, n) for n in st["lens"]))
    t = ends - span + torch.arange(span, device="cuda")                      # [B, span]: every token that some query of the sequence sees
    far = (ends - m + torch.arange(m, device="cuda")).unsqueeze(2) - t.unsqueeze(1)   # [B, m, span]
    s = torch.einsum("bmgrd,btgd->bgrmt", q.float().view(B, m, G, H // G, D), tokens_of(st["k"], t)) * D ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].view(G, H // G, 1, 1) * far.float()[:, None, None]
    seen = (far >= 0) & (t >= 0).unsqueeze(1) & (far < (c["window"] or span + m))
    s = torch.where(seen[:, None, None], s, -torch.inf)
    most = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(most), 0.0, most))
    total = e.sum(-1, keepdim=True)
    o = torch.einsum("bgrmt,btgd->bmgrd", e / torch.where(total > 0, total, 1.0), tokens_of(st["v"], t))
    return o.reshape(B * m, H * D).to(q.dtype)


def plain_write(st):
    c, got = st["c"], []
    who = torch.arange(c["B"], device="cuda").unsqueeze(1)
    at = torch.tensor(st["lens"], device="cuda").unsqueeze(1) + torch.arange(c["m"], device="cuda")
    for which, new, bits in (("k", st["rows"][0], c["kb"]), ("v", st["rows"][1], c["vb"])):
        for held, t in zip(st[which], quantise(new, bits, c["D"])):
            held[who, at] = t.view(c["B"], c["m"], c["G"], -1)
        got.append(tokens_of(st[which], at).to(new.dtype))
    return got


def plain_read(st):
    c = st["c"]
    inside = torch.arange(capacity(c), device="cuda") < torch.tensor(st["lens"], device="cuda").unsqueeze(1)
    return [torch.where(inside[..., None, None], values(*st[which]), 0.0).to(DTYPES[c["dtype"]]) for which in "kv"]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    st, c = state, state["c"]
    if not own:
        return {"attend": plain_attend, "write": plain_write, "read": plain_read}[c["kind"]](st)
    gpu, ctx, cache = st["gpu"], st["ctx"], st["cache"]
    gpu.batch_begin(ctx)
    if c["kind"] == "attend":
        gpu.attention_with_quant_cache(ctx, cache, 0, st["rows"][0], st["out"], tokens=c["m"], softcap=c["softcap"], window=c["window"],
                                       slopes=st["slopes"])
        result = st["out"].buffer
    elif c["kind"] == "write":
        # (the rows stay "pending": the lengths do not move, so the next pass writes the same places)
        gpu.quant_cache_update(ctx, cache, 0, *st["rows"], tokens=c["m"], advance=False)
        result = [gpu.quant_cache_gather(ctx, cache, 0, which, length=c["m"], last=True, pending=c["m"]) for which in "kv"]
    else:
        result = [gpu.quant_cache_gather(ctx, cache, 0, which) for which in "kv"]
    gpu.batch_commit(ctx)
    return result


def row_bytes(c, which):
    return c["D"] * c[which + "b"] // 8 + c["D"] // GROUP * 2


def visible(c, n):
    """Tokens of a sequence of n that any of its queries sees."""
    return min(n, c["window"] + c["m"] - 1) if c["window"] else n


def work(case):
    c, es = case, 4 if case["dtype"] == "f32" else 2
    mean = (c["lo"] + c["hi"]) / 2
    row = row_bytes(c, "k") + row_bytes(c, "v")
    if c["kind"] == "attend":
        # lengths are uniform in lo .. hi: the mean of what a window leaves, from a few of them
        some = [visible(c, c["lo"] + (c["hi"] - c["lo"]) * i / 64) for i in range(65)]
        seen = sum(some) / len(some)
        return dict(bytes=c["B"] * (seen * c["G"] * row + 2 * c["m"] * c["H"] * c["D"] * es),
                    flops=4.0 * c["B"] * c["m"] * c["H"] * c["D"] * seen)
    wide = c["G"] * c["D"] * es * 2
    if c["kind"] == "write":  # rows in, codes and scales out; codes and scales in, values out
        n = c["B"] * c["m"]
        return dict(bytes=n * 2 * (wide + c["G"] * row), flops=4.0 * n * 2 * c["G"] * c["D"])
    return dict(bytes=c["B"] * (mean * c["G"] * row + capacity(c) * wide), flops=c["B"] * mean * 2 * c["G"] * c["D"])


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def held64(x, bits):
    """Values in float64 that a cache holds for x [..., D]."""
    top = 7.0 if bits == 4 else 127.0
    g = x.double().unflatten(-1, (-1, GROUP))
    most = g.abs().max(dim=-1, keepdim=True).values
    scale = (most / torch.full_like(most, top)).to(torch.bfloat16).double()
    code = torch.round(g / scale)
    code = torch.minimum(torch.maximum(torch.where(scale == 0, torch.zeros_like(code), code), -torch.full_like(code, top)),
                         torch.full_like(code, top))
    return (code * scale).flatten(-2)


def exact(case, seed):
    c = case
    B, G, D, T = c["B"], c["G"], c["D"], capacity(c)
    lens = lengths(c, seed)
    if c["kind"] == "write":
        return [held64(x.view(B, c["m"], G, D), bits) for x, bits in zip(rows_in(c, seed), (c["kb"], c["vb"]))]
    if c["kind"] == "read":
        got = []
        for which, bits in (("k", c["kb"]), ("v", c["vb"])):
            x = held64(history(c, seed, which).view(B, T, G, D), bits)
            got.append(torch.where((torch.arange(T, device="cuda")[None, :] < torch.tensor(lens, device="cuda")[:, None])[..., None, None],
                                   x, torch.zeros((), dtype=torch.float64, device="cuda")))
        return got
    m, H = c["m"], c["H"]
    K, V, (q,) = history(c, seed, "k").view(B, T, G, D), history(c, seed, "v").view(B, T, G, D), rows_in(c, seed)
    q = q.view(B, m, H, D).double()
    slopes = slopes_of(c)
    out = torch.zeros((B, m, H, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        first = 0 if not c["window"] else max(0, n - m - c["window"] + 1)
        place = torch.arange(n - m, n, device="cuda", dtype=torch.float64)
        far = place[:, None] - torch.arange(first, n, device="cuda", dtype=torch.float64)[None, :]
        hidden = far < 0
        if c["window"]:
            hidden = hidden | (far >= c["window"])
        for g in range(G):
            heads = slice(g * (H // G), (g + 1) * (H // G))
            k, v = held64(K[b, first:n, g], c["kb"]), held64(V[b, first:n, g], c["vb"])
            s = q[b, :, heads].reshape(-1, D) @ k.T / math.sqrt(D)
            if c["softcap"]:
                s = torch.tanh(s / c["softcap"]) * c["softcap"]
            s = s.view(m, H // G, -1)
            if slopes is not None:
                s = s - slopes[heads].double()[None, :, None] * far[:, None, :]
            s = s.masked_fill(hidden[:, None, :], -math.inf)
            w = torch.softmax(s, dim=-1).masked_fill(hidden.all(dim=1)[:, None, None], 0.0)
            out[b, :, heads] = (w.reshape(-1, w.shape[-1]) @ v).view(m, H // G, D)
    return out.view(B * m, H * D)
