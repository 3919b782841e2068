"""The calls of a serving step at their limits: scores of any size, lengths and block numbers out of range, threads with heads of different sizes, results joined in
passes."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import hologram_b200 as hb
from serving_step_reference import HALF_STEP, attend
from test_serving_step_gpu import test_block_cache_attention as attention_case
from test_serving_step_gpu import CACHE_WEIGHT_HALF, TORCH, WEIGHT_HALF, Cache, attention, check, f64, packed, starts_of, strided

pytestmark = pytest.mark.gpu


# ---- scores of any size ------------------------------------------------------------------------------------------------


def winners(codes, limits, sign, v, half, dtype):
    """Scores are `codes` (whole numbers) times a factor that is large, its sign `sign`: a row's result is the mean of v [n, vdim] over the keys with
    its largest score. All of those have the same score to the last bit, and the next score is lower by the factor at least: 46 and more powers
    of two. Off by: the stored type's half step; a weight's rounding; 2^-18 for exponentials, the logarithm of a scale and the sums in f32;
    and what the other keys' weights, 2^-46 of the largest each at most, bring in."""
    out, off = np.zeros((len(limits), v.shape[1])), np.zeros((len(limits), v.shape[1]))
    for i, e in enumerate(limits):
        c = codes[:e] * sign[i]
        top = c == c.max()
        out[i] = v[:e][top].mean(0)
        off[i] = 1.1 * (HALF_STEP[dtype] * np.abs(out[i]) + (half + 2.0 ** -18) * np.abs(v[:e][top]).mean(0) + e * 2.0 ** -46 * np.abs(v[:e]).max())
    return out, off


# the factor of the scores is 2^(power - 3) log2(e): from 46 steps a code to far beyond what f32 tells apart from its neighbours
POWERS = [8, 12, 20, 26, 60]


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("dtype,block,dim,new", [
    ("bf16", 16, 64, [70, 40]), ("f16", 32, 128, [70, 40]), ("bf16", 48, 80, [300]),       # portions on the tensor cores
    ("bf16", 24, 64, [70, 40]), ("f32", 16, 64, [70, 40]), ("f16", 24, 128, [130]),        # portions of odd blocks, of f32
    ("bf16", 16, 64, [1, 1]), ("f16", 24, 128, [2, 1]), ("f32", 16, 128, [1, 1]),          # few rows
    ("bf16", 16, 40, [3, 1]),                                                              # any shape
])
def test_block_cache_attention_of_scores_of_any_size(backend, dtype, block, dim, new, power):
    """Query rows with one value of 1 or -1, key scales of 1: a score is a code times the call's scale."""
    rng = np.random.default_rng(19)
    cache = Cache(rng, [n + 260 for n in new], block, 1, dim, dim)
    cache.host["k_scales"][:] = 1.0
    cache.dev["k_scales"].fill_(1.0)
    starts, rows = starts_of(new), sum(new)
    sign, column = rng.choice([-1.0, 1.0], (rows, 2)), rng.integers(0, dim, (rows, 2))
    q = torch.zeros(rows, 2, dim)
    for r in range(rows):
        for h in range(2):
            q[r, h, column[r, h]] = sign[r, h]
    q, out = q.reshape(rows, 2 * dim).to(TORCH[dtype]).cuda(), torch.zeros(rows, 2 * dim, dtype=TORCH[dtype], device="cuda")
    attention(backend, cache, q, starts, out, 2, dtype, scale=2.0 ** (power - 3))
    backend.synchronize()
    got = f64(out).reshape(rows, 2, dim)
    for s, n in enumerate(cache.lens):
        k, v = cache.held("k", s, n)[:, 0], cache.held("v", s, n)[:, 0]
        for i in range(new[s]):
            for h in range(2):
                r = int(starts[s]) + i
                want, off = winners(k[:, column[r, h]], [n - new[s] + 1 + i], [sign[r, h]], v, CACHE_WEIGHT_HALF[dtype], dtype)
                check(got[r:r + 1, h], want, off, f"row {r} head {h}")


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f16", 128), ("bf16", 80), ("f32", 64), ("bf16", 40)])
def test_packed_attention_of_scores_of_any_size(backend, dtype, dim, power):
    """As over the cache: keys of whole numbers of at most 7 bits, which all types hold."""
    rng = np.random.default_rng(20)
    lens = [300, 40, 150]
    starts, rows = starts_of(lens), sum(lens)
    sign, column = rng.choice([-1.0, 1.0], (rows, 2)), rng.integers(0, dim, (rows, 2))
    q = torch.zeros(rows, 2, dim)
    for r in range(rows):
        for h in range(2):
            q[r, h, column[r, h]] = sign[r, h]
    q = q.reshape(rows, 2 * dim).to(TORCH[dtype]).cuda()
    k = torch.from_numpy(rng.integers(-127, 128, (rows, dim)).astype(np.float32)).to(TORCH[dtype]).cuda()
    v, out = strided(rng, rows, dim, dim, dtype), torch.zeros(rows, 2 * dim, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, starts, out, 2, 1, dim, dim, True, dtype, scale=2.0 ** (power - 3))
    backend.synchronize()
    got, kf, vf = f64(out).reshape(rows, 2, dim), f64(k), f64(v)
    for a, b in zip(starts, starts[1:]):
        for r in range(a, b):
            for h in range(2):
                want, off = winners(kf[a:b, column[r, h]], [r + 1 - a], [sign[r, h]], vf[a:b], WEIGHT_HALF[dtype], dtype)
                check(got[r:r + 1, h], want, off, f"row {r} head {h}")


# ---- lengths and block numbers out of range ----------------------------------------------------------------------------


@pytest.mark.parametrize("what", ["nothing", "negative", "short", "long", "block", "no block"])
@pytest.mark.parametrize("dtype,block,dim,new", [
    ("bf16", 16, 64, [40, 37, 50]), ("f16", 24, 64, [40, 37, 50]), ("f32", 16, 64, [40, 37, 50]),      # portions: tensor cores, odd blocks, f32
    ("bf16", 32, 64, [1, 1, 1]), ("f32", 16, 128, [2, 3, 1]), ("f16", 24, 64, [1, 3, 2]),              # few rows
    ("bf16", 16, 40, [2, 3, 1]), ("f32", 8, 33, [20, 30, 10]),                                         # any shape
])
def test_what_is_out_of_range_counts_the_same_in_every_shape(backend, what, dtype, block, dim, new):
    """Reported, and: a length counts as 0 below and as the table's positions above, rows that see nothing are zero, a block that does not
    exist holds zeros."""
    rng = np.random.default_rng(21)
    cache = Cache(rng, [90, 110, 130], block, 2, dim, dim)
    starts, rows = starts_of(new), sum(new)
    q, out = strided(rng, rows, 4 * dim, 4 * dim, dtype), torch.full((rows, 4 * dim), 5.0, dtype=TORCH[dtype], device="cuda")
    k, v = [[cache.held(p, s, n) for s, n in enumerate(cache.lens)] for p in "kv"]
    length = cache.lens[1]
    if what in ("block", "no block"):
        cache.table[1, 1] = cache.blocks if what == "block" else -1
        for x in (k[1], v[1]):
            x[block:2 * block] = 0
    elif what == "long":
        # every block of the table is one of the cache's, so that only the length is wrong
        cache.table[cache.table < 0] = 0
        length = cache.width * block
        k[1], v[1] = cache.held("k", 1, length), cache.held("v", 1, length)
        cache.lens[1] = length + 9
    else:
        cache.lens[1] = {"nothing": 0, "negative": -4, "short": new[1] // 2}[what]
        length = max(cache.lens[1], 0)
    attention(backend, cache, q, starts, out, 4, dtype)
    with pytest.raises(hb.BackendError, match="out of range"):
        backend.synchronize()
    backend.synchronize()
    got, qf = f64(out).reshape(rows, 4, dim), f64(q).reshape(rows, 4, dim)
    for s, n in enumerate([cache.lens[0], length, cache.lens[2]]):
        a, b = int(starts[s]), int(starts[s + 1])
        for h in range(4):
            want, off = attend(qf[a:b, h], k[s][:, h // 2], v[s][:, h // 2], n - (b - a) + 1 + np.arange(b - a), dim ** -0.5, dtype, CACHE_WEIGHT_HALF[dtype])
            check(got[a:b, h], want, off, f"sequence {s}")


# ---- threads -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("large,small", [((112, 128), (80, 80)), ((48, 64), (16, 16)), ((240, 256), (144, 144))])
@pytest.mark.parametrize("new", [[1, 1], [2, 1]])
def test_threads_with_heads_of_different_sizes(large, small, new):
    """Two threads, a context each, whose calls want different amounts of shared memory of one kernel: the smaller one's takes nothing from the
    larger one's."""
    def make(dims, seed):
        be, rng = hb.B200Backend(0), np.random.default_rng(seed)
        dim, vdim = dims
        cache = Cache(rng, [300, 77], 16, 2, dim, vdim)
        q, out = strided(rng, sum(new), 4 * dim, 4 * dim, "bf16"), torch.zeros(sum(new), 4 * vdim, dtype=torch.bfloat16, device="cuda")
        return be, cache, q, out

    def run(made):
        be, cache, q, out = made
        out.zero_()
        kept = attention(be, cache, q, starts_of(new), out, 4, "bf16")
        be.synchronize()
        got, starts = f64(out).reshape(sum(new), 4, cache.vdim), starts_of(new)
        for s, n in enumerate(cache.lens):
            a, b = int(starts[s]), int(starts[s + 1])
            k, v = cache.held("k", s, n), cache.held("v", s, n)
            for h in range(4):
                want, off = attend(f64(q).reshape(-1, 4, cache.dim)[a:b, h], k[:, h // 2], v[:, h // 2], n - (b - a) + 1 + np.arange(b - a), cache.dim ** -0.5, "bf16",
                                   CACHE_WEIGHT_HALF["bf16"])
                check(got[a:b, h], want, off, f"sequence {s}")
        del kept

    with ThreadPoolExecutor(1) as one, ThreadPoolExecutor(1) as other:
        first, second = one.submit(make, large, 41).result(), other.submit(make, small, 42).result()
        try:
            for _ in range(2):
                one.submit(run, first).result()
                other.submit(run, second).result()
        finally:
            one.submit(first[0].close).result()
            other.submit(second[0].close).result()


# ---- eight rows of 128 columns -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new,before,block,heads,kv", [
    ([1] * 40, [(37 * i) % 300 for i in range(40)], 32, 16, 2),      # whole planes, one after another in a CTA
    ([1, 1, 1], [900, 0, 2500], 16, 12, 2),                          # six rows of eight, parts of planes joined
    ([2, 3, 1, 0, 4], [70, 5, 640, 3, 1000], 24, 8, 4),
    ([1], [3999], 64, 8, 1),
])
def test_results_of_eight_rows_are_joined_in_two_passes(backend, new, before, block, heads, kv, dtype):
    attention_case(backend, new, before, block, heads, kv, 128, 128, dtype)
