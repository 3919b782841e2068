"""The calls of a serving step over several sequences against 64 bits: PackedAttention, BlockCacheWrite, BlockCacheAttention, LogitRules."""
import numpy as np
import pytest
import torch

import hologram_b200 as hb
from hologram_b200 import kernel_call as kc
from serving_step_reference import HALF_STEP, attend, rules, write_plane

pytestmark = pytest.mark.gpu
rb = kc.rb
TAG = {"bf16": kc.DTYPE_BF16, "f16": kc.DTYPE_F16, "f32": kc.DTYPE_F32}
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# rounding of the weights of a softmax where they go through the tensor core: bf16 and f16 as they are, f32 as two f16 terms
WEIGHT_HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -21}
CACHE_WEIGHT_HALF = {"bf16": 2.0 ** -11, "f16": 2.0 ** -11, "f32": 2.0 ** -21}


class Slots:
    """A device workspace whose slots are torch tensors."""

    def __init__(self, backend, n=12):
        self.ws, self.n, self.kept = hb.DeviceWorkspace(backend, n), 0, []

    def __call__(self, tensor):
        if tensor is None:
            return kc.NONE
        torch.cuda.synchronize()          # made on torch's stream, read on the backend's
        storage = tensor.untyped_storage()
        at = tensor.storage_offset() * tensor.element_size()
        self.ws.bind(self.n, storage.data_ptr(), storage.nbytes())
        self.kept.append(tensor)
        self.n += 1
        return rb(self.n - 1, at, storage.nbytes() - at)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def f64(tensor):
    return tensor.double().cpu().numpy()


def starts_of(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int64)


def strided(rng, rows, width, ld, dtype, offset=0, sigma=1.0):
    """[rows, width] of pitch `ld` inside a larger buffer of other values."""
    flat = torch.from_numpy(rng.standard_normal(offset + rows * ld + 8).astype(np.float32) * sigma).to(TORCH[dtype]).cuda()
    return flat[offset:offset + rows * ld].view(rows, ld)[:, :width]


def check(got, want, off, what=""):
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), f"{what}: {bad.sum()} values off, the worst {np.max(np.abs(got - want)[bad])} at a bound of {off[bad].min()}, first {np.argwhere(bad)[0]}"


# ---- packed attention --------------------------------------------------------------------------------------------------


def packed(backend, q, k, v, starts, out, heads, kv, dim, vdim, causal, dtype, scale=0):
    s = Slots(backend)
    rows = q.shape[0]
    call = kc.PackedAttentionCall(s(q), s(k), s(v), s(i32(list(map(int, starts)))), s(out), rows, len(starts) - 1, heads, kv, dim, vdim, q.stride(0), k.stride(0), v.stride(0),
                                  out.stride(0), kc.f32_bits(scale) if scale else 0, int(causal), TAG[dtype])
    backend.dispatch(kc.KernelCall.PackedAttention(call), s.ws)
    return s


def packed_reference(q, k, v, starts, heads, kv, dim, vdim, causal, dtype, scale=0):
    q, k, v = f64(q).reshape(-1, heads, dim), f64(k).reshape(-1, kv, dim), f64(v).reshape(-1, kv, vdim)
    out, off = np.full((q.shape[0], heads, vdim), np.nan), np.zeros((q.shape[0], heads, vdim))
    for a, b in zip(starts, starts[1:]):
        for h in range(heads):
            g = h // (heads // kv)
            limits = np.arange(1, b - a + 1) if causal else np.full(b - a, b - a)
            out[a:b, h], off[a:b, h] = attend(q[a:b, h], k[a:b, g], v[a:b, g], limits, scale or dim ** -0.5, dtype, WEIGHT_HALF[dtype])
    return out.reshape(q.shape[0], -1), off.reshape(q.shape[0], -1)


PACKED = [
    # lens, heads, kv_heads, dim, vdim, causal
    ([1], 1, 1, 16, 16, True),
    ([1, 1, 1], 4, 2, 64, 64, True),
    ([0, 5, 0, 0, 130, 1, 0], 4, 1, 64, 64, True),
    ([127, 1, 128, 129], 2, 2, 128, 128, True),
    ([300, 17, 64], 6, 2, 80, 80, True),
    ([255, 257], 4, 4, 128, 64, False),
    ([33, 200, 9, 77, 140], 8, 2, 48, 112, False),
    ([513], 2, 1, 128, 128, True),
    ([40, 3], 3, 3, 20, 12, True),       # dims that no tile takes
    ([21, 90], 2, 1, 256, 512, False),   # dims beyond the tiles
    ([2] * 150, 2, 2, 64, 64, True),     # more sequences in a tile than warps
    ([700, 640], 2, 1, 128, 128, True),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens,heads,kv,dim,vdim,causal", PACKED)
def test_packed_attention(backend, lens, heads, kv, dim, vdim, causal, dtype):
    rng = np.random.default_rng(sum(lens) * 131 + dim)
    starts = starts_of(lens)
    rows = int(starts[-1])
    q, k, v = strided(rng, rows, heads * dim, heads * dim, dtype), strided(rng, rows, kv * dim, kv * dim, dtype), strided(rng, rows, kv * vdim, kv * vdim, dtype)
    out = torch.full((rows, heads * vdim), 7.0, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, starts, out, heads, kv, dim, vdim, causal, dtype)
    backend.synchronize()
    want, off = packed_reference(q, k, v, starts, heads, kv, dim, vdim, causal, dtype)
    check(f64(out), want, off)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("pad,offset", [(8, 8), (24, 0), (1, 0), (0, 1), (3, 5)])
def test_packed_attention_strides_and_rows_of_nobody(backend, dtype, pad, offset):
    """Pitches wider than the rows, operands that begin off a 16-byte boundary, rows before the first and behind the last sequence."""
    rng = np.random.default_rng(pad * 10 + offset)
    heads, kv, dim, rows, starts = 4, 2, 64, 230, np.array([3, 70, 70, 211])
    q, k, v = (strided(rng, rows, n * dim, n * dim + pad, dtype, offset) for n in (heads, kv, kv))
    flat = torch.full((offset + rows * (heads * dim + pad) + 8,), 5.0, dtype=TORCH[dtype], device="cuda")
    out = flat[offset:offset + rows * (heads * dim + pad)].view(rows, -1)[:, :heads * dim]
    packed(backend, q, k, v, starts, out, heads, kv, dim, dim, True, dtype)
    backend.synchronize()
    want, off = packed_reference(q, k, v, starts, heads, kv, dim, dim, True, dtype)
    got = f64(out)
    check(got[3:211], want[3:211], off[3:211])
    assert np.all(got[:3] == 5.0) and np.all(got[211:] == 5.0)
    whole = f64(flat)
    assert np.all(whole[:offset] == 5.0) and np.all(whole[offset + rows * (heads * dim + pad):] == 5.0)
    if pad:
        assert np.all(whole[offset:offset + rows * (heads * dim + pad)].reshape(rows, -1)[:, heads * dim:] == 5.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_packed_attention_keeps_what_is_not_finite_to_the_rows_that_see_it(backend, dtype, causal, poison):
    rng = np.random.default_rng(5)
    heads, kv, dim, starts = 4, 2, 64, np.array([0, 50, 60, 190, 400])
    rows = 400
    q, k, v = (strided(rng, rows, n * dim, n * dim, dtype) for n in (heads, kv, kv))
    want, off = packed_reference(q, k, v, starts, heads, kv, dim, dim, causal, dtype)
    v[55, 3] = poison          # a value of the second sequence, one of the last one, a key of the third, a query of the first
    v[300, 70] = poison
    k[100, 5] = poison
    q[20, 2] = poison
    out = torch.zeros(rows, heads * dim, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, starts, out, heads, kv, dim, dim, causal, dtype)
    backend.synchronize()
    got = f64(out)
    clean = np.ones((rows, heads, dim), dtype=bool)
    clean[(55 if causal else 50):60, :2, 3] = False
    clean[(300 if causal else 190 + 0):400, 2:, 6] = False
    if not causal:
        clean[190:400, 2:, 6] = False
    clean[(100 if causal else 60):190, :2] = False
    clean[20, 0] = False
    clean = clean.reshape(rows, -1)
    check(got[clean], want[clean], off[clean])
    spoilt = got.reshape(rows, heads, dim)
    assert not np.isfinite(spoilt[55 if causal else 50:60, :2, 3]).any() and not np.isfinite(spoilt[300:400, 2:, 6]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_packed_attention_of_extreme_scores(backend, dtype):
    """Scores far apart, all alike, and rows whose scores are all -inf."""
    rng = np.random.default_rng(9)
    heads, kv, dim, starts = 2, 1, 64, np.array([0, 150, 280, 290])
    q, k, v = (strided(rng, 290, n * dim, n * dim, dtype) for n in (heads, kv, kv))
    q[:150] *= 40
    k[150:280] = 0
    k[280:290] = 0
    k[280:290, 0] = -float("inf")
    q[280:290] = 0.5
    out = torch.zeros(290, heads * dim, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, starts, out, heads, kv, dim, dim, True, dtype)
    backend.synchronize()
    want, off = packed_reference(q[:280], k[:280], v[:280], starts[:3], heads, kv, dim, dim, True, dtype)
    check(f64(out)[:280], want, off)
    assert np.all(f64(out)[280:] == 0)


def test_packed_attention_long_sequence_repeats_bit_for_bit(backend):
    rng = np.random.default_rng(3)
    heads, kv, dim, lens = 8, 2, 128, [2100, 5, 900, 1]
    starts = starts_of(lens)
    rows = int(starts[-1])
    q, k, v = (strided(rng, rows, n * dim, n * dim, "bf16") for n in (heads, kv, kv))
    outs = [torch.zeros(rows, heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    for o in outs:
        packed(backend, q, k, v, starts, o, heads, kv, dim, dim, True, "bf16")
    backend.synchronize()
    assert all(torch.equal(outs[0].view(torch.int16), o.view(torch.int16)) for o in outs)
    pick = np.array([0, 1, 127, 128, 1000, 2099, 2100, 2104, 2105, 2500, 3004, 3005])
    qf, kf, vf = f64(q).reshape(rows, heads, dim), f64(k).reshape(rows, kv, dim), f64(v).reshape(rows, kv, dim)
    for r in pick:
        s = int(np.searchsorted(starts, r, side="right")) - 1
        a = int(starts[s])
        for h in (0, 5):
            want, off = attend(qf[r:r + 1, h], kf[a:r + 1, h // 4], vf[a:r + 1, h // 4], [r + 1 - a], dim ** -0.5, "bf16", WEIGHT_HALF["bf16"])
            check(f64(outs[0])[r:r + 1, h * dim:(h + 1) * dim], want, off, f"row {r}")


@pytest.mark.parametrize("starts", [[0, 50, 40, 100], [-3, 50, 100], [0, 50, 101], [0, 2 ** 31 - 1, 100], [100, 0, 50]])
def test_packed_attention_reports_bad_starts(backend, starts):
    rng = np.random.default_rng(1)
    for dtype, dim in (("bf16", 64), ("f32", 64), ("bf16", 20)):
        q, k, v = (strided(rng, 100, n * dim, n * dim, dtype) for n in (2, 1, 1))
        out = torch.zeros(100, 2 * dim, dtype=TORCH[dtype], device="cuda")
        packed(backend, q, k, v, starts, out, 2, 1, dim, dim, True, dtype)
        with pytest.raises(hb.BackendError, match="out of range"):
            backend.synchronize()
        backend.synchronize()


# ---- the block cache ---------------------------------------------------------------------------------------------------


class Cache:
    def __init__(self, rng, lens, block, kv, dim, vdim, extra=2, sigma=1.0):
        self.block, self.kv, self.dim, self.vdim, self.lens = block, kv, dim, vdim, list(lens)
        need = [-(-n // block) for n in lens]
        self.blocks, self.width = sum(need) + extra, max(1, max(need)) + 1
        order = list(rng.permutation(self.blocks))
        table = np.full((len(lens), self.width), -1, dtype=np.int32)
        for s, n in enumerate(need):
            for j in range(n):
                table[s, j] = order.pop()
        self.host = {"k_codes": rng.integers(-127, 128, (self.blocks, kv, block, dim)).astype(np.int8), "v_codes": rng.integers(-127, 128, (self.blocks, kv, block, vdim)).astype(np.int8),
                     "k_scales": (np.exp(rng.standard_normal((self.blocks, kv)) * 0.5) * sigma / 60).astype(np.float32),
                     "v_scales": (np.exp(rng.standard_normal((self.blocks, kv)) * 0.5) / 60).astype(np.float32)}
        self.table = table
        self.dev = {n: torch.from_numpy(a.copy()).cuda() for n, a in self.host.items()}

    def refs(self, s, starts):
        return [s(None if starts is None else i32(list(map(int, starts)))), s(i32(self.lens)), s(torch.from_numpy(self.table.copy()).cuda())] + [
            s(self.dev[n]) for n in ("k_codes", "k_scales", "v_codes", "v_scales")]

    def held(self, which, s, n):
        """The values of sequence s's first n positions [n, kv, dim]."""
        out = np.zeros((n, self.kv, self.dim if which == "k" else self.vdim))
        for p in range(n):
            b = self.table[s, p // self.block]
            out[p] = self.host[which + "_codes"][b, :, p % self.block].astype(np.float64) * self.host[which + "_scales"][b].astype(np.float64)[:, None]
        return out


def write(backend, cache, k, v, starts, dtype):
    s = Slots(backend)
    call = kc.BlockCacheWriteCall(s(k), s(v), *cache.refs(s, starts), k.shape[0], len(cache.lens), cache.kv, cache.dim, cache.vdim, k.stride(0), v.stride(0), cache.block,
                                  cache.blocks, cache.width, TAG[dtype])
    backend.dispatch(kc.KernelCall.BlockCacheWrite(call), s.ws)
    return s


def attention(backend, cache, q, starts, out, heads, dtype, scale=0):
    s = Slots(backend)
    call = kc.BlockCacheAttentionCall(s(q), *cache.refs(s, starts), s(out), q.shape[0], len(cache.lens), heads, cache.kv, cache.dim, cache.vdim, q.stride(0), out.stride(0),
                                      cache.block, cache.blocks, cache.width, kc.f32_bits(scale) if scale else 0, TAG[dtype])
    backend.dispatch(kc.KernelCall.BlockCacheAttention(call), s.ws)
    return s


def same_cache(cache):
    for name, want in cache.host.items():
        got = cache.dev[name].cpu().numpy()
        if name.endswith("scales"):
            got, want = got.view(np.uint32), want.view(np.uint32)
        bad = np.argwhere(got != want)
        assert not len(bad), f"{name}: {len(bad)} differ, first {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


WRITES = [
    # new rows, positions before, block, kv_heads, dim, vdim
    ([1], [0], 16, 1, 64, 64),
    ([1, 1, 1, 1], [0, 15, 16, 100], 16, 2, 128, 128),
    ([40, 0, 7, 33], [5, 3, 0, 31], 32, 2, 64, 128),
    ([300, 1], [0, 64], 64, 3, 80, 48),
    ([17, 64], [63, 1], 128, 1, 20, 12),
    ([5, 9, 2], [2, 0, 4], 1, 2, 16, 16),
    ([100], [1000], 24, 2, 40, 33),
    ([3, 2000], [1021, 0], 1024, 1, 16, 16),
    ([13] * 30, list(range(0, 300, 10)), 16, 1, 256, 512),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new,before,block,kv,dim,vdim", WRITES)
def test_block_cache_write(backend, new, before, block, kv, dim, vdim, dtype):
    rng = np.random.default_rng(sum(new) + block)
    cache = Cache(rng, [a + b for a, b in zip(new, before)], block, kv, dim, vdim)
    starts = starts_of(new)
    rows = int(starts[-1])
    for turn in range(2):       # the second turn writes the same rows again: nothing changes
        k, v = strided(rng, rows, kv * dim, kv * dim + 8, dtype), strided(rng, rows, kv * vdim, kv * vdim, dtype, sigma=3.0)
        write(backend, cache, k, v, starts, dtype)
        write(backend, cache, k, v, starts, dtype)
        backend.synchronize()
        write_plane(f64(k).reshape(rows, kv, dim), cache.host["k_codes"], cache.host["k_scales"], starts, cache.lens, cache.table, block)
        write_plane(f64(v).reshape(rows, kv, vdim), cache.host["v_codes"], cache.host["v_scales"], starts, cache.lens, cache.table, block)
        same_cache(cache)


def test_block_cache_write_single_rows_without_starts(backend):
    rng = np.random.default_rng(2)
    cache = Cache(rng, [1, 40, 17, 16, 33], 16, 2, 64, 64)
    for turn in range(20):
        k, v = (strided(rng, 5, 128, 128, "bf16", sigma=2.0 ** turn) for _ in range(2))
        write(backend, cache, k, v, None, "bf16")
        backend.synchronize()
        for p, x in (("k", k), ("v", v)):
            write_plane(f64(x).reshape(5, 2, 64), cache.host[p + "_codes"], cache.host[p + "_scales"], np.arange(6), cache.lens, cache.table, 16)
        same_cache(cache)
        cache.lens = [min(n + 1, (cache.width - 1) * 16) for n in cache.lens]
        need = [-(-n // 16) for n in cache.lens]
        if any(cache.table[s, n - 1] < 0 for s, n in enumerate(need)):
            break


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_block_cache_write_of_special_values(backend, dtype):
    """Zero rows, values that are not finite, subnormal scales, the largest values, quotients that end in a half."""
    rng = np.random.default_rng(8)
    cache = Cache(rng, [16] * 8, 16, 1, 32, 32)
    rows = 8 * 16
    x = rng.standard_normal((rows, 32)).astype(np.float32)
    x[:16] = 0
    x[16, 3], x[17, 4], x[18, 5] = np.nan, np.inf, -np.inf
    x[32:48] = np.nan
    tiny = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}[dtype]
    x[48:64] = rng.integers(-200, 201, (16, 32)) * tiny
    x[64:80] = np.clip(x[64:80], -1, 1) * {"bf16": 3e38, "f16": 6e4, "f32": 3.4e38}[dtype]
    x[80:96] = rng.integers(-254, 255, (16, 32)) / 2.0
    x[80, 0] = 127.0
    x[96:112] = rng.integers(-3, 4, (16, 32)) * 0.5
    x[112:128] = np.inf
    t = torch.from_numpy(x).to(TORCH[dtype]).cuda()
    write(backend, cache, t, t, starts_of([16] * 8), dtype)
    backend.synchronize()
    for p in "kv":
        write_plane(f64(t).reshape(rows, 1, 32), cache.host[p + "_codes"], cache.host[p + "_scales"], starts_of([16] * 8), cache.lens, cache.table, 16)
    same_cache(cache)


CACHES = [
    # new rows, positions before, block, heads, kv_heads, dim, vdim
    ([1], [0], 16, 1, 1, 64, 64),
    ([1, 1, 1, 1, 1], [0, 15, 16, 100, 333], 16, 8, 2, 128, 128),
    ([1, 1, 1], [511, 2, 1030], 32, 32, 8, 128, 128),
    ([1] * 9, [5, 77, 200, 31, 32, 33, 0, 640, 1], 64, 12, 2, 64, 64),
    ([3, 0, 5, 1], [100, 9, 0, 64], 32, 4, 4, 96, 48),
    ([40, 17], [0, 333], 128, 8, 1, 128, 128),
    ([100, 1, 300], [29, 1000, 0], 32, 4, 2, 128, 128),
    ([5, 9, 2], [2, 0, 4], 1, 4, 2, 16, 32),
    ([7, 1], [100, 77], 24, 6, 2, 40, 33),
    ([1, 2], [1500, 90], 1024, 16, 1, 256, 256),
    ([1, 4], [300, 3], 48, 20, 1, 80, 512),
    ([1], [5000], 16, 16, 2, 128, 128),
    ([64], [700], 16, 48, 2, 64, 128),
    # portions: many rows of a sequence
    ([200, 5, 70], [1000, 0, 333], 64, 8, 2, 96, 48),
    ([130], [0], 16, 4, 4, 64, 64),
    ([33, 257, 0, 80], [129, 64, 7, 1500], 48, 6, 2, 80, 112),
    ([90, 31], [37, 600], 24, 4, 1, 128, 128),      # blocks that are no multiple of 16 rows
    ([1, 300, 1, 1], [2000, 5, 0, 127], 32, 8, 1, 128, 64),
    ([128], [2944], 128, 4, 1, 16, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new,before,block,heads,kv,dim,vdim", CACHES)
def test_block_cache_attention(backend, new, before, block, heads, kv, dim, vdim, dtype):
    rng = np.random.default_rng(sum(before) + dim)
    cache = Cache(rng, [a + b for a, b in zip(new, before)], block, kv, dim, vdim)
    starts = starts_of(new)
    rows = int(starts[-1])
    q = strided(rng, rows, heads * dim, heads * dim, dtype)
    out = torch.full((rows, heads * vdim), 7.0, dtype=TORCH[dtype], device="cuda")
    for _ in range(2):
        attention(backend, cache, q, None if all(n == 1 for n in new) else starts, out, heads, dtype)
    backend.synchronize()
    got, qf = f64(out).reshape(rows, heads, vdim), f64(q).reshape(rows, heads, dim)
    for s, n in enumerate(cache.lens):
        k, v = cache.held("k", s, n), cache.held("v", s, n)
        a, m = int(starts[s]), new[s]
        for h in range(heads):
            g = h // (heads // kv)
            want, off = attend(qf[a:a + m, h], k[:, g], v[:, g], n - m + 1 + np.arange(m), dim ** -0.5, dtype, CACHE_WEIGHT_HALF[dtype])
            check(got[a:a + m, h], want, off, f"sequence {s} head {h}")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("pad,offset", [(8, 8), (1, 0), (3, 5)])
def test_block_cache_attention_strides_and_rows_of_nobody(backend, dtype, pad, offset):
    rng = np.random.default_rng(4)
    cache = Cache(rng, [20, 0, 7], 16, 2, 64, 64)
    heads, rows, starts = 4, 12, np.array([2, 5, 5, 9])
    q = strided(rng, rows, 256, 256 + pad, dtype, offset)
    flat = torch.full((offset + rows * (256 + pad) + 8,), 5.0, dtype=TORCH[dtype], device="cuda")
    out = flat[offset:offset + rows * (256 + pad)].view(rows, -1)[:, :256]
    attention(backend, cache, q, starts, out, heads, dtype, scale=0.3)
    backend.synchronize()
    got, qf = f64(out), f64(q).reshape(rows, heads, 64)
    for s, n in ((0, 20), (2, 7)):
        k, v = cache.held("k", s, n), cache.held("v", s, n)
        a, b = int(starts[s]), int(starts[s + 1])
        for h in range(heads):
            want, off = attend(qf[a:b, h], k[:, h // 2], v[:, h // 2], n - (b - a) + 1 + np.arange(b - a), float(np.float32(0.3)), dtype, CACHE_WEIGHT_HALF[dtype])
            check(got[a:b, 64 * h:64 * h + 64], want, off)
    assert np.all(got[:2] == 5.0) and np.all(got[9:] == 5.0)
    whole = f64(flat)
    assert np.all(whole[:offset] == 5.0) and np.all(whole[offset + rows * (256 + pad):] == 5.0)
    assert np.all(whole[offset:offset + rows * (256 + pad)].reshape(rows, -1)[:, 256:] == 5.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_block_cache_attention_of_queries_of_any_size(backend, dtype):
    """Rows whose largest value is tiny or huge, rows of zeros, rows with one value that is not finite."""
    rng = np.random.default_rng(6)
    cache = Cache(rng, [70] * 8, 32, 1, 64, 64)
    q = strided(rng, 8, 128, 128, dtype)
    q[0] *= 1e-4
    q[1] *= 200.0
    q[2] = 0
    q[3, 5] *= 1000.0
    q[4, :64] *= 1e-3
    q[5, 7] = float("nan")
    q[6, 7] = float("inf")
    out = torch.zeros(8, 128, dtype=TORCH[dtype], device="cuda")
    attention(backend, cache, q, None, out, 2, dtype)
    backend.synchronize()
    got, qf = f64(out).reshape(8, 2, 64), f64(q).reshape(8, 2, 64)
    for s in range(8):
        k, v = cache.held("k", s, 70)[:, 0], cache.held("v", s, 70)[:, 0]
        for h in range(2):
            if not np.isfinite(qf[s, h]).all():
                assert not np.isfinite(got[s, h]).any()
                continue
            want, off = attend(qf[s:s + 1, h], k, v, [70], 0.125, dtype, CACHE_WEIGHT_HALF[dtype])
            check(got[s:s + 1, h], want, off, f"sequence {s} head {h}")


def test_block_cache_attention_keeps_stale_rows_and_blocks_out(backend):
    """Scales of blocks that nobody has, and what stands behind a sequence's last position, reach no result; blocks may be shared."""
    rng = np.random.default_rng(7)
    cache = Cache(rng, [50, 50, 33], 16, 2, 128, 128, extra=4)
    cache.table[1, :3] = cache.table[0, :3]        # full blocks that two sequences share
    used = set(int(b) for s, n in enumerate(cache.lens) for b in cache.table[s, :-(-n // 16)])
    for b in range(cache.blocks):
        if b not in used:
            cache.host["k_scales"][b] = cache.host["v_scales"][b] = np.nan
    cache.dev = {n: torch.from_numpy(a.copy()).cuda() for n, a in cache.host.items()}
    q = strided(rng, 3, 1024, 1024, "bf16")
    out = torch.zeros(3, 1024, dtype=torch.bfloat16, device="cuda")
    attention(backend, cache, q, None, out, 8, "bf16")
    backend.synchronize()
    first = out.clone()
    for s, n in enumerate(cache.lens):
        b = cache.table[s, n // 16]
        for p in "kv":
            cache.dev[p + "_codes"][int(b), :, n % 16:] = 127
    attention(backend, cache, q, None, out, 8, "bf16")
    backend.synchronize()
    assert torch.equal(first, out)
    qf = f64(q).reshape(3, 8, 128)
    for s, n in enumerate(cache.lens):
        k, v = cache.held("k", s, n), cache.held("v", s, n)
        for h in range(8):
            want, off = attend(qf[s:s + 1, h], k[:, h // 4], v[:, h // 4], [n], 128 ** -0.5, "bf16", CACHE_WEIGHT_HALF["bf16"])
            check(f64(out).reshape(3, 8, 128)[s:s + 1, h], want, off)


@pytest.mark.parametrize("what", ["block", "negative", "length", "short", "starts"])
def test_block_cache_reports_bad_tables(backend, what):
    rng = np.random.default_rng(11)
    for dim in (64, 40):
        cache = Cache(rng, [40, 40, 40], 16, 2, dim, dim)
        starts = [0, 2, 3, 6]
        if what == "block":
            cache.table[1, 2] = cache.blocks
        elif what == "negative":
            cache.table[1, 2] = -1
        elif what == "length":
            cache.lens[1] = cache.width * 16 + 1
        elif what == "short":
            cache.lens[2] = 2
        else:
            starts = [0, 4, 3, 6]
        q, k, v = strided(rng, 6, 4 * dim, 4 * dim, "bf16"), strided(rng, 6, 2 * dim, 2 * dim, "bf16"), strided(rng, 6, 2 * dim, 2 * dim, "bf16")
        out = torch.zeros(6, 4 * dim, dtype=torch.bfloat16, device="cuda")
        write(backend, cache, k, v, starts, "bf16")
        with pytest.raises(hb.BackendError, match="out of range"):
            backend.synchronize()
        attention(backend, cache, q, starts, out, 4, "bf16")
        with pytest.raises(hb.BackendError, match="out of range"):
            backend.synchronize()
        backend.synchronize()


@pytest.mark.parametrize("dtype,block", [("bf16", 16), ("f16", 24), ("f32", 16)])
@pytest.mark.parametrize("what", ["block", "negative", "length", "short", "starts"])
def test_block_cache_reports_bad_tables_of_portions(backend, what, dtype, block):
    """As above where a sequence has many rows; what is not wrong is as it would be without the mistake."""
    rng = np.random.default_rng(16)
    cache = Cache(rng, [300, 280, 310], block, 2, 64, 64)
    starts = [0, 70, 110, 200]
    q = strided(rng, 200, 256, 256, dtype)
    out = torch.zeros(200, 256, dtype=TORCH[dtype], device="cuda")
    qf, want = f64(q).reshape(200, 4, 64), {}
    for s, n in ((0, 300), (2, 310)):
        a, b = starts[s], starts[s + 1]
        k, v = cache.held("k", s, n), cache.held("v", s, n)
        for h in range(4):
            want[s, h] = attend(qf[a:b, h], k[:, h // 2], v[:, h // 2], n - (b - a) + 1 + np.arange(b - a), 0.125, dtype, CACHE_WEIGHT_HALF[dtype])
    if what == "block":
        cache.table[1, 7] = cache.blocks
    elif what == "negative":
        cache.table[1, 0] = -7
    elif what == "length":
        cache.lens[1] = cache.width * block + 1
    elif what == "short":
        cache.lens[1] = 12
    else:
        starts = [0, 70, 60, 200]
    attention(backend, cache, q, starts, out, 4, dtype)
    with pytest.raises(hb.BackendError, match="out of range"):
        backend.synchronize()
    backend.synchronize()
    got = f64(out).reshape(200, 4, 64)
    for h in range(4):
        check(got[:60, h], want[0, h][0][:60], want[0, h][1][:60], "sequence 0")      # the 60 rows that are nobody else's
        if what != "starts":
            check(got[110:, h], *want[2, h], "sequence 2")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_portions_with_queries_of_any_size(backend, dtype):
    """Among the rows of a portion: zeros, tiny and huge ones, one value that stands out, one that is not finite; the others take no notice."""
    rng = np.random.default_rng(17)
    cache = Cache(rng, [200, 90], 16, 1, 64, 64)
    q = strided(rng, 130, 128, 128, dtype)
    q[0] *= 1e-4
    q[1] *= 200.0
    q[2] = 0
    q[3, 5] *= 1000.0
    q[4, :64] *= 1e-3
    q[70, 7] = float("nan")
    q[101, 70] = float("-inf")
    out, starts = torch.zeros(130, 128, dtype=TORCH[dtype], device="cuda"), [0, 80, 130]
    attention(backend, cache, q, starts, out, 2, dtype)
    backend.synchronize()
    got, qf = f64(out).reshape(130, 2, 64), f64(q).reshape(130, 2, 64)
    for s, n in enumerate(cache.lens):
        k, v = cache.held("k", s, n)[:, 0], cache.held("v", s, n)[:, 0]
        for i in range(starts[s], starts[s + 1]):
            for h in range(2):
                if not np.isfinite(qf[i, h]).all():
                    assert not np.isfinite(got[i, h]).any()
                    continue
                want, off = attend(qf[i:i + 1, h], k, v, [n - (starts[s + 1] - 1 - i)], 0.125, dtype, CACHE_WEIGHT_HALF[dtype])
                check(got[i:i + 1, h], want, off, f"row {i} head {h}")


# ---- logit rules -------------------------------------------------------------------------------------------------------


RULES = [
    # rows, vocabulary, history, biases of a row, masks
    (1, 1, 1, 0, False),
    (1, 131, 40, 3, True),
    (3, 1000, 300, 7, True),
    (5, 8192, 64, 0, True),
    (2, 8193, 1, 1, False),
    (4, 32000, 5000, 300, True),
    (2, 70001, 2000, 11, True),
    (70, 517, 33, 5, True),
    (1, 300007, 9000, 20, True),
]


def apply_rules(backend, z, out, history=None, spans=None, params=None, bias=None, masks=None, mask_of=None, dtype="f32"):
    s = Slots(backend)
    starts, ids, values = bias if bias is not None else (None, None, None)
    call = kc.LogitRulesCall(s(z), s(history), s(spans), s(params), s(starts), s(ids), s(values), s(masks), s(mask_of), s(out), z.shape[0], z.shape[1], z.stride(0), out.stride(0),
                             0 if history is None else history.shape[1], 0 if ids is None else ids.numel(), 0 if masks is None else masks.shape[0],
                             0 if masks is None else masks.shape[1], TAG[dtype])
    backend.dispatch(kc.KernelCall.LogitRules(call), s.ws)
    return s


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,length,biases,masked", RULES)
@pytest.mark.parametrize("in_place", [False, True])
def test_logit_rules(backend, rows, vocab, length, biases, masked, in_place, dtype):
    rng = np.random.default_rng(vocab + rows)
    z = strided(rng, rows, vocab, vocab + 3 * in_place, dtype, offset=in_place, sigma=4.0)
    history = rng.integers(0, vocab, (rows, length)).astype(np.int32)
    history[:, ::3] = rng.integers(0, min(vocab, 20), history[:, ::3].shape)
    history[:, 1::7] = np.where(rng.random(history[:, 1::7].shape) < 0.5, -1, vocab)      # ids outside the vocabulary
    total = rng.integers(0, length + 1, rows)
    total[0] = length
    spans = np.stack([rng.integers(0, total + 1), total], 1).astype(np.int32)
    params = np.stack([rng.choice([1.0, 1.2, 0.8], rows), rng.choice([0.0, 0.5, -0.3], rows), rng.choice([0.0, 0.25], rows), rng.choice([0.0, 1.0, 0.6], rows)], 1).astype(np.float32)
    counts = rng.integers(0, biases + 1, rows)
    counts[0] = biases
    starts = starts_of(counts)
    ids = rng.integers(-1, vocab + 1, max(1, int(starts[-1]))).astype(np.int32)           # tokens named twice among them
    values = rng.standard_normal(ids.size).astype(np.float32)
    words = (vocab + 31) // 32 + 1
    masks = rng.integers(0, 2 ** 32, (3, words), dtype=np.uint64).astype(np.uint32)
    mask_of = rng.integers(-1, 3, rows).astype(np.int32)
    zf = f64(z)
    out = z if in_place else torch.zeros(rows, vocab + 5, dtype=TORCH[dtype], device="cuda")[:, :vocab]
    apply_rules(backend, z, out, torch.from_numpy(history).cuda(), torch.from_numpy(spans).cuda(), torch.from_numpy(params).cuda(),
                (i32(starts.tolist()), torch.from_numpy(ids).cuda(), torch.from_numpy(values).cuda()) if biases else None,
                torch.from_numpy(masks.view(np.int32)).cuda() if masked else None, torch.from_numpy(mask_of).cuda() if masked else None, dtype)
    backend.synchronize()
    got = f64(out)
    for r in range(rows):
        allowed = ((masks[mask_of[r]][np.arange(vocab) >> 5] >> (np.arange(vocab) & 31).astype(np.uint32)) & 1).astype(bool) if masked and mask_of[r] >= 0 else None
        want, off = rules(zf[r], history[r].tolist(), spans[r], params[r], list(zip(ids[starts[r]:starts[r + 1]].tolist(), values[starts[r]:starts[r + 1]])) if biases else [], allowed)
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(got[r]))
        check(got[r][fine], want[fine], off[fine] * 1.01 + HALF_STEP[dtype] * np.abs(want[fine]) * 1.01 + (2.0 ** -25 if dtype == "f16" else 0.0), f"row {r}")


def test_logit_rules_each_alone(backend):
    """Every operand may be absent; without any the logits are copied."""
    rng = np.random.default_rng(12)
    z = strided(rng, 3, 777, 777, "f32")
    zf, out = f64(z), torch.zeros(3, 777, device="cuda")
    apply_rules(backend, z, out)
    backend.synchronize()
    assert np.array_equal(f64(out), zf)
    params = torch.tensor([[5.0, 5.0, 5.0, 0.5]] * 3, device="cuda")
    apply_rules(backend, z, out, params=params)
    backend.synchronize()
    assert np.array_equal(f64(out), zf * 2)
    masks = torch.zeros(3, 25, dtype=torch.int32, device="cuda")
    masks[1] = -1
    apply_rules(backend, z, out, masks=masks)
    backend.synchronize()
    assert np.all(f64(out)[[0, 2]] == -np.inf) and np.array_equal(f64(out)[1], zf[1])
    apply_rules(backend, z, out, bias=(i32([0, 0, 2, 2]), i32([5, 5]), torch.tensor([1.0, 3.0], device="cuda")))
    backend.synchronize()
    zf[1, 5] = np.float32(zf[1, 5]) + np.float32(3.0)
    assert np.array_equal(f64(out), zf)


def test_logit_rules_of_more_rows_than_a_grid_is_high(backend):
    rng = np.random.default_rng(15)
    z = strided(rng, 70000, 33, 33, "f32")
    out = torch.zeros(70000, 33, device="cuda")
    history = torch.from_numpy(rng.integers(0, 33, (70000, 3)).astype(np.int32)).cuda()
    masks = torch.full((70000, 2), -1, dtype=torch.int32, device="cuda")
    masks[:, 1] = torch.arange(70000, device="cuda") & 1                      # odd rows may choose token 32
    bias = i32(np.minimum(np.arange(70001), 69999).tolist()), torch.zeros(69999, dtype=torch.int32, device="cuda"), torch.arange(69999, dtype=torch.float32, device="cuda")
    apply_rules(backend, z, out, history, i32([[0, 3]]).repeat(70000, 1), torch.tensor([[1.0, 0.5, 0.0, 0.0]], device="cuda").repeat(70000, 1), bias, masks)
    backend.synchronize()
    want = f64(z)
    forbidden = np.arange(70000) % 2 == 0
    assert np.all(np.isneginf(f64(out)[forbidden, 32])) and np.isfinite(f64(out)[~forbidden, 32]).all()
    # row r has r added to its token 0, the last row nothing: another rounding of numbers up to r
    first, more = f64(out)[:, 0], np.where(np.arange(70000) < 69999, np.arange(70000), 0)
    seen = (history.cpu().numpy() == 0).any(1)
    assert np.all(np.abs(first - (want[:, 0] - 0.5 * seen + more)) <= 2.0 ** -24 * (2 * np.abs(want[:, 0]) + 1 + 2 * more))
    out[:, 0], out[:, 32], z[:, 0], z[:, 32] = 0, 0, 0, 0
    want, history = f64(z), history.clone()
    history[(history == 0) | (history == 32)] = -1
    seen = np.zeros((70000, 33), dtype=bool)
    for column in history.cpu().numpy().T:
        seen[np.arange(70000)[column >= 0], column[column >= 0]] = True
    # a difference with 0.5 in f32: one rounding of a value
    assert np.all(np.abs(f64(out) - (want - 0.5 * seen)) <= 2.0 ** -24 * (np.abs(want) + 0.5))


@pytest.mark.parametrize("what", ["spans", "total", "bias", "mask"])
def test_logit_rules_report_bad_numbers(backend, what):
    z, out = torch.zeros(2, 100, device="cuda"), torch.zeros(2, 100, device="cuda")
    history, spans, params = torch.zeros(2, 10, dtype=torch.int32, device="cuda"), i32([[0, 10], [0, 10]]), torch.ones(2, 4, device="cuda")
    bias = (i32([0, 1, 2]), i32([1, 2]), torch.ones(2, device="cuda"))
    masks, mask_of = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), i32([0, 1])
    if what == "spans":
        spans[1, 0] = 11
    elif what == "total":
        spans[1, 1] = 11
    elif what == "bias":
        bias[0][2] = 3
    else:
        mask_of[1] = 2
    apply_rules(backend, z, out, history, spans, params, bias, masks, mask_of)
    with pytest.raises(hb.BackendError, match="out of range"):
        backend.synchronize()
    backend.synchronize()


# ---- refusals ----------------------------------------------------------------------------------------------------------


def refused(backend, slots, call, variant):
    with pytest.raises(hb.BackendError) as e:
        backend.dispatch(call, slots.ws)
    assert e.value.variant == variant
    backend.synchronize()


def test_refusals_of_packed_attention(backend):
    bf = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")
    base = dict(rows=10, sequences=2, heads=4, kv_heads=2, dim=64, vdim=64, q_ld=256, k_ld=128, v_ld=128, ld=256, scale_bits=0, causal=1, dtype=kc.DTYPE_BF16)
    for change, variant in (({"dtype": kc.DTYPE_I8}, "UnsupportedOp"), ({"kv_heads": 3}, "UnsupportedOp"), ({"kv_heads": 0}, "UnsupportedOp"), ({"dim": 0}, "ShapeMismatch"),
                            ({"dim": 513, "q_ld": 4 * 513, "k_ld": 2 * 513}, "ShapeMismatch"), ({"q_ld": 255}, "ShapeMismatch"), ({"ld": 255}, "ShapeMismatch"),
                            ({"rows": 11}, "SlotOutOfRange"), ({"sequences": 3}, "SlotOutOfRange"), ({"scale_bits": kc.f32_bits(-1.0)}, "UnsupportedOp"),
                            ({"scale_bits": kc.f32_bits(float("nan"))}, "UnsupportedOp"), ({"scale_bits": kc.f32_bits(float("inf"))}, "UnsupportedOp")):
        s = Slots(backend)
        refs = [s(bf(10, 256)), s(bf(10, 128)), s(bf(10, 128)), s(i32([0, 4, 10])), s(bf(10, 256))]
        refused(backend, s, kc.KernelCall.PackedAttention(kc.PackedAttentionCall(*refs, *dict(base, **change).values())), variant)
    s = Slots(backend)
    q = s(bf(10, 256))
    call = kc.PackedAttentionCall(q, s(bf(10, 128)), s(bf(10, 128)), s(i32([0, 4, 10])), q, *base.values())
    refused(backend, s, kc.KernelCall.PackedAttention(call), "SlotOutOfRange")          # the output over an input
    # nothing to do is no error
    s = Slots(backend)
    refs = [s(bf(10, 256)), s(bf(10, 128)), s(bf(10, 128)), s(i32([0, 4, 10])), s(bf(10, 256))]
    for none in ({"rows": 0}, {"sequences": 0}, {"heads": 0}):
        backend.dispatch(kc.KernelCall.PackedAttention(kc.PackedAttentionCall(*refs, *dict(base, **none).values())), s.ws)
    backend.synchronize()


def test_refusals_of_the_block_cache(backend):
    rng = np.random.default_rng(1)
    cache = Cache(rng, [20, 30], 16, 2, 64, 64)
    bf = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")
    sizes = dict(rows=5, sequences=2, kv_heads=2, dim=64, vdim=64, k_ld=128, v_ld=128, block_rows=16, blocks=cache.blocks, table_ld=cache.width, dtype=kc.DTYPE_BF16)
    for change, variant in (({"dtype": kc.DTYPE_I32}, "UnsupportedOp"), ({"kv_heads": 0}, "ShapeMismatch"), ({"block_rows": 0}, "ShapeMismatch"), ({"block_rows": 1025}, "ShapeMismatch"),
                            ({"blocks": 0}, "ShapeMismatch"), ({"blocks": cache.blocks + 1}, "SlotOutOfRange"), ({"table_ld": 0}, "ShapeMismatch"),
                            ({"table_ld": cache.width + 1}, "SlotOutOfRange"), ({"k_ld": 127}, "ShapeMismatch"), ({"rows": 6}, "SlotOutOfRange"), ({"dim": 513}, "ShapeMismatch")):
        s = Slots(backend)
        call = kc.BlockCacheWriteCall(s(bf(5, 128)), s(bf(5, 128)), *cache.refs(s, [0, 2, 5]), *dict(sizes, **change).values())
        refused(backend, s, kc.KernelCall.BlockCacheWrite(call), variant)
    s = Slots(backend)
    refs = cache.refs(s, [0, 2, 5])
    refs[5] = refs[3]           # one buffer for the codes of keys and values
    refused(backend, s, kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(s(bf(5, 128)), s(bf(5, 128)), *refs, *sizes.values())), "SlotOutOfRange")
    sizes = dict(rows=5, sequences=2, heads=4, kv_heads=2, dim=64, vdim=64, q_ld=256, ld=256, block_rows=16, blocks=cache.blocks, table_ld=cache.width, scale_bits=0, dtype=kc.DTYPE_BF16)
    for change, variant in (({"heads": 5}, "UnsupportedOp"), ({"q_ld": 200}, "ShapeMismatch"), ({"ld": 200}, "ShapeMismatch"), ({"vdim": 0}, "ShapeMismatch"),
                            ({"scale_bits": kc.f32_bits(-0.5)}, "UnsupportedOp"), ({"sequences": 3}, "SlotOutOfRange"), ({"dtype": kc.DTYPE_I8}, "UnsupportedOp")):
        s = Slots(backend)
        call = kc.BlockCacheAttentionCall(s(bf(5, 256)), *cache.refs(s, [0, 2, 5]), s(bf(5, 256)), *dict(sizes, **change).values())
        refused(backend, s, kc.KernelCall.BlockCacheAttention(call), variant)
    s = Slots(backend)          # without starts every sequence has one row
    call = kc.BlockCacheAttentionCall(s(bf(5, 256)), *cache.refs(s, None), s(bf(5, 256)), *sizes.values())
    refused(backend, s, kc.KernelCall.BlockCacheAttention(call), "ShapeMismatch")


def test_refusals_of_logit_rules(backend):
    f = lambda *shape: torch.zeros(*shape, device="cuda")
    n = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")

    def call(drop=(), change=None, **over):
        s = Slots(backend)
        ops = {"logits": f(2, 100), "history": n(2, 10), "spans": n(2, 2), "params": f(2, 4), "bias_starts": n(3), "bias_ids": n(4), "bias_values": f(4), "masks": n(2, 4), "mask_of": n(2),
               "output": f(2, 100)}
        ops.update(over)
        sizes = dict(rows=2, vocab=100, ld=100, out_ld=100, history_ld=10, biases=4, mask_rows=2, mask_ld=4, dtype=kc.DTYPE_F32)
        sizes.update(change or {})
        return s, kc.KernelCall.LogitRules(kc.LogitRulesCall(*[s(None if k in drop else t) for k, t in ops.items()], *sizes.values()))

    for drop in ("spans", "params", "history", "bias_starts", "bias_values", "bias_ids"):
        refused(backend, *call((drop,)), "UnsupportedOp")
    refused(backend, *call(("masks",)), "UnsupportedOp")
    for change in ({"mask_ld": 3}, {"history_ld": 0}, {"biases": 0}, {"mask_rows": 0}, {"ld": 99}):
        refused(backend, *call(change=change), "ShapeMismatch")
    refused(backend, *call(("mask_of",), {"mask_rows": 1}), "ShapeMismatch")
    for change in ({"rows": 3}, {"history_ld": 11}, {"biases": 5}, {"mask_rows": 3}):
        refused(backend, *call(change=change), "SlotOutOfRange")
    refused(backend, *call(change={"dtype": kc.DTYPE_I32}), "UnsupportedOp")


def test_sizes_whose_bytes_pass_64_bits_are_refused(backend):
    """Products of sizes that come out small modulo 2^64 are as far outside the buffers as they look."""
    rng = np.random.default_rng(1)
    cache, s = Cache(rng, [20], 16, 1, 64, 64), Slots(backend, 30)
    small = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")
    refs, k, v, q, o = cache.refs(s, None), s(small(1, 64)), s(small(1, 64)), s(small(1, 64)), s(small(1, 64))
    # 2^31 blocks of 1024 rows for 2^20 heads of 512 columns: 2^70 bytes
    sizes = dict(rows=1, sequences=1, kv_heads=2 ** 20, dim=512, vdim=512, k_ld=2 ** 29, v_ld=2 ** 29, block_rows=1024, blocks=2 ** 31 - 1, table_ld=2, dtype=kc.DTYPE_BF16)
    refused(backend, s, kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(k, v, *refs, *sizes.values())), "ShapeMismatch")
    sizes = dict(rows=1, sequences=1, heads=2 ** 20, kv_heads=2 ** 20, dim=512, vdim=512, q_ld=2 ** 29, ld=2 ** 29, block_rows=1024, blocks=2 ** 31 - 1, table_ld=2, scale_bits=0, dtype=kc.DTYPE_BF16)
    refused(backend, s, kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(q, *refs, o, *sizes.values())), "ShapeMismatch")
    z, n = s(torch.zeros(64, device="cuda")), s(torch.zeros(64, dtype=torch.int32, device="cuda"))
    out = s(torch.zeros(64, device="cuda"))
    # masks of 2^62 words; a history of 2^62 tokens; logits of 2^62 + 2^31 tokens less 2^31
    for change, of in (({"mask_rows": 2 ** 31, "mask_ld": 2 ** 31}, "masks"), ({"rows": 2 ** 31 - 1, "history_ld": 2 ** 31 - 1, "ld": 1, "out_ld": 1, "vocab": 1}, "history"),
                       ({"rows": 2 ** 30 + 1, "ld": 2 ** 32 - 1, "out_ld": 2 ** 32 - 1, "vocab": 2 ** 30}, "logits")):
        call = dict(rows=1, vocab=64, ld=64, out_ld=64, history_ld=4, biases=0, mask_rows=1, mask_ld=2, dtype=kc.DTYPE_F32)
        call.update(change)
        ops = {"logits": z, "history": n if of == "history" else kc.NONE, "spans": n if of == "history" else kc.NONE, "params": z if of == "history" else kc.NONE, "bias_starts": kc.NONE,
               "bias_ids": kc.NONE, "bias_values": kc.NONE, "masks": n if of == "masks" else kc.NONE, "mask_of": n if of == "masks" else kc.NONE, "output": out}
        refused(backend, s, kc.KernelCall.LogitRules(kc.LogitRulesCall(*ops.values(), *call.values())), "SlotOutOfRange")


def test_no_host_workspace_form(backend):
    host = hb.HostWorkspace([np.zeros(4096, dtype=np.uint8) for _ in range(10)])
    for call in (kc.KernelCall.PackedAttention(kc.PackedAttentionCall()), kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall()),
                 kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall()), kc.KernelCall.LogitRules(kc.LogitRulesCall())):
        with pytest.raises(hb.BackendError, match="no host-workspace form"):
            backend.dispatch(call, host)


# ---- the calls together, and what a caller may do around them ----------------------------------------------------------


class Step:
    """A step of several sequences: the rows' attention, their keys and values into the cache, and rules on logits, which here are the
    attention's output of a row read as a vocabulary. `prompts` (packed attention) before the cache has anything, then single tokens."""

    def __init__(self, rng, dtype, new, before, heads=8, kv=2, dim=64, block=16):
        self.dtype, self.heads, self.kv, self.dim, self.new = dtype, heads, kv, dim, new
        self.starts, rows, self.vocab = starts_of(new), int(sum(new)), heads * dim
        self.before, self.after = before, [a + b for a, b in zip(new, before)]
        self.qkv = strided(rng, rows, (heads + 2 * kv) * dim, (heads + 2 * kv) * dim, dtype)       # one product's columns
        self.q, self.k, self.v = self.qkv[:, :heads * dim], self.qkv[:, heads * dim:(heads + kv) * dim], self.qkv[:, (heads + kv) * dim:]
        self.out = torch.zeros(rows, self.vocab, dtype=TORCH[dtype], device="cuda")
        self.history = rng.integers(0, self.vocab, (rows, 12)).astype(np.int32)
        self.params = np.tile(np.array([[1.25, 0.5, 0.25, 0.5]], dtype=np.float32), (rows, 1))
        self.masks = rng.integers(0, 2 ** 32, (rows, self.vocab // 32), dtype=np.uint64).astype(np.uint32)
        self.logits = torch.zeros(rows, self.vocab, dtype=TORCH[dtype], device="cuda")
        self.rule_args = [torch.from_numpy(self.history).cuda(), i32([[4, 12]] * rows), torch.from_numpy(self.params).cuda()]
        self.dev_masks = torch.from_numpy(self.masks.view(np.int32)).cuda()

    def calls(self, s, cache, prompt):
        """The step's calls over the slots `s`, the cache's lengths being those after the step."""
        rows, bare = self.q.shape[0], kc.NONE
        starts = s(i32(list(map(int, self.starts)))) if prompt else None
        q, k, v, out = s(self.q), s(self.k), s(self.v), s(self.out)
        refs = cache.refs(s, None)
        if prompt:
            refs[0] = starts
        sizes = (rows, len(self.new), self.kv, self.dim, self.dim, self.k.stride(0), self.v.stride(0), cache.block, cache.blocks, cache.width, TAG[self.dtype])
        calls = [kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(k, v, *refs, *sizes))]
        if prompt:
            calls.append(kc.KernelCall.PackedAttention(kc.PackedAttentionCall(q, k, v, starts, out, rows, len(self.new), self.heads, self.kv, self.dim, self.dim, self.q.stride(0),
                                                                              self.k.stride(0), self.v.stride(0), self.vocab, 0, 1, TAG[self.dtype])))
        else:
            calls.append(kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(q, *refs, out, rows, len(self.new), self.heads, self.kv, self.dim, self.dim, self.q.stride(0),
                                                                                      self.vocab, cache.block, cache.blocks, cache.width, 0, TAG[self.dtype])))
        history, spans, params = (s(t) for t in self.rule_args)
        calls.append(kc.KernelCall.LogitRules(kc.LogitRulesCall(out, history, spans, params, bare, bare, bare, s(self.dev_masks), bare, s(self.logits), rows, self.vocab, self.vocab,
                                                                self.vocab, 12, 0, rows, self.vocab // 32, TAG[self.dtype])))
        return calls

    def check(self, cache, prompt):
        """After the calls: the cache code for code, every row's logits within their bounds."""
        rows, d = self.q.shape[0], self.dim
        kf, vf = f64(self.k).reshape(rows, self.kv, d), f64(self.v).reshape(rows, self.kv, d)
        write_plane(kf, cache.host["k_codes"], cache.host["k_scales"], self.starts, self.after, cache.table, cache.block)
        write_plane(vf, cache.host["v_codes"], cache.host["v_scales"], self.starts, self.after, cache.table, cache.block)
        same_cache(cache)
        qf, got = f64(self.q).reshape(rows, self.heads, d), f64(self.logits)
        for s, n in enumerate(self.after):
            a, m = int(self.starts[s]), self.new[s]
            k, v = (kf[a:a + m], vf[a:a + m]) if prompt else (cache.held("k", s, n), cache.held("v", s, n))
            parts = [attend(qf[a:a + m, h], k[:, h // (self.heads // self.kv)], v[:, h // (self.heads // self.kv)], n - m + 1 + np.arange(m), d ** -0.5, self.dtype,
                            (WEIGHT_HALF if prompt else CACHE_WEIGHT_HALF)[self.dtype]) for h in range(self.heads)]
            for i in range(m):
                z, z_off = (np.concatenate([p[part][i] for p in parts]) for part in (0, 1))
                allowed = (self.masks[a + i][np.arange(self.vocab) >> 5] >> (np.arange(self.vocab) & 31).astype(np.uint32) & 1).astype(bool)
                want, off = rules(z, self.history[a + i], (4, 12), self.params[a + i], [], allowed)
                fine = np.isfinite(want)
                assert np.array_equal(fine, np.isfinite(got[a + i]))
                # an error of the attention's grows by the repetition's 1.25 and the temperature's 1 / 0.5 at most
                check(got[a + i][fine], want[fine], (2.5 * z_off + 1.01 * off + HALF_STEP[self.dtype] * (np.abs(want) + 2.5 * z_off))[fine] + (2.0 ** -25 if self.dtype == "f16" else 0.0), f"row {a + i}")


def serve(rng, dtype, dispatch, backend):
    """Prompts of four sequences, then three single tokens of each: everything of a step is enqueued before anything is read."""
    lens, block = [37, 1, 130, 16], 16
    cache = Cache(rng, [n + 3 for n in lens], block, 2, 64, 64)
    results = []
    for turn in range(4):
        new = lens if turn == 0 else [1] * 4
        step = Step(rng, dtype, new, [0] * 4 if turn == 0 else [n + turn - 1 for n in lens], block=block)
        cache.lens = step.after
        s = Slots(backend, 24)
        dispatch(step.calls(s, cache, turn == 0), s)
        backend.synchronize()
        step.check(cache, turn == 0)
        results.append(step.logits.clone())
    return results


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_a_served_batch_of_prompts_and_tokens(backend, dtype):
    def dispatch(calls, s):
        for c in calls:
            backend.dispatch(c, s.ws)

    serve(np.random.default_rng(21), dtype, dispatch, backend)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_served_batch_recorded_and_replayed(dtype):
    """The same steps as graphs on another stream, each replayed twice: the calls write the same values again."""
    be, stream = hb.B200Backend(0), torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    kept = []

    def direct(calls, s):
        for c in calls:
            be.dispatch(c, s.ws)

    def recorded(calls, s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            for c in calls:
                be.dispatch(c, s.ws)
        with torch.cuda.stream(stream):
            graph.replay()
            graph.replay()
        stream.synchronize()
        kept.append((graph, s))

    first = serve(np.random.default_rng(22), dtype, direct, be)
    second = serve(np.random.default_rng(22), dtype, recorded, be)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    for graph, s in kept:
        s.ws.close()
    del graph
    kept.clear()
    be.close()


def test_the_first_call_that_needs_a_buffer_is_not_recorded():
    be, stream, rng = hb.B200Backend(0), torch.cuda.Stream(), np.random.default_rng(1)
    be.set_stream(stream.cuda_stream)
    for new in ([1, 1], [100, 40]):
        cache = Cache(rng, [200, 100], 16, 2, 64, 64)
        q, out = strided(rng, sum(new), 256, 256, "bf16"), torch.zeros(sum(new), 256, dtype=torch.bfloat16, device="cuda")
        s = Slots(be, 12)
        call = kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(s(q), *cache.refs(s, starts_of(new)), s(out), sum(new), 2, 4, 2, 64, 64, 256, 256, 16, cache.blocks, cache.width, 0,
                                                                            kc.DTYPE_BF16))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            with pytest.raises(hb.BackendError, match="first call") as e:
                be.dispatch(call, s.ws)
        assert e.value.variant == "Dispatch"
        del e           # its traceback holds the workspace, which must not go in the middle of the next recording
        be.dispatch(call, s.ws)
        be.synchronize()
        del graph
        graph = torch.cuda.CUDAGraph()
        want = out.clone()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            be.dispatch(call, s.ws)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del graph
    be.close()


def archive_of(calls_of, tensors, outputs):
    """A `.holo` image of `calls_of(slot references)` whose slots are input ports of the tensors' sizes, those of `outputs` output ports."""
    from hologram_b200 import holo
    w = holo.HoloWriter()
    names = list(tensors)
    refs = {n: kc.rb(i) for i, n in enumerate(names)}
    w.calls.extend(calls_of(refs))
    kinds = {torch.bfloat16: kc.DTYPE_BF16, torch.float16: kc.DTYPE_F16, torch.float32: kc.DTYPE_F32, torch.int32: kc.DTYPE_I32, torch.int8: kc.DTYPE_I8}
    for i, n in enumerate(names):
        t = tensors[n]
        (w.outputs if n in outputs else w.inputs).append(holo.Port(n, i, t.numel(), kinds[t.dtype], list(t.shape)))
    w.exec_plan = [[i] for i in range(len(w.calls))]
    w.slot_bytes = [t.numel() * t.element_size() for t in tensors.values()]
    return w.finish()


def test_the_calls_through_an_archive_session(backend):
    """One archive of write, attention and rules; walked, then recorded and replayed: the dispatched calls' bits. Addressed sessions refuse them."""
    rng = np.random.default_rng(23)
    rows, lens = 3, [20, 65, 1]
    cache = Cache(rng, lens, 16, 2, 64, 64)
    step = Step(rng, "bf16", [1] * 3, [n - 1 for n in lens])
    tensors = {"q": step.q.contiguous(), "k": step.k.contiguous(), "v": step.v.contiguous(), "lengths": i32(lens), "table": torch.from_numpy(cache.table).cuda(),
               **{n: cache.dev[n].clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales")}, "history": step.rule_args[0], "spans": step.rule_args[1], "params": step.rule_args[2],
               "masks": step.dev_masks, "out": step.out, "logits": step.logits}

    def calls(r):
        planes = [kc.NONE, r["lengths"], r["table"], r["k_codes"], r["k_scales"], r["v_codes"], r["v_scales"]]
        return [kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(r["k"], r["v"], *planes, rows, rows, 2, 64, 64, 128, 128, 16, cache.blocks, cache.width, kc.DTYPE_BF16)),
                kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(r["q"], *planes, r["out"], rows, rows, 8, 2, 64, 64, 512, 512, 16, cache.blocks, cache.width, 0, kc.DTYPE_BF16)),
                kc.KernelCall.LogitRules(kc.LogitRulesCall(r["out"], r["history"], r["spans"], r["params"], kc.NONE, kc.NONE, kc.NONE, r["masks"], kc.NONE, r["logits"], rows, 512, 512, 512,
                                                           12, 0, rows, 16, kc.DTYPE_BF16))]

    image = archive_of(calls, tensors, ("out", "logits"))
    s = Slots(backend, 24)
    for c in step.calls(s, cache, False):
        backend.dispatch(c, s.ws)
    backend.synchronize()
    step.check(cache, False)
    bits = lambda t: t.cpu().contiguous().view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()
    session = hb.InferenceSession(backend, image)
    for n, t in tensors.items():
        if n not in ("out", "logits"):
            session.write(n, bits(t))
    session.execute()
    assert np.array_equal(session.read("logits", np.int16).reshape(rows, 512), bits(step.logits))
    session.capture()
    session.execute()
    assert np.array_equal(session.read("logits", np.int16).reshape(rows, 512), bits(step.logits))
    assert np.array_equal(session.read("k_codes", np.int8).reshape(cache.host["k_codes"].shape), cache.host["k_codes"])
    session.close()
    with pytest.raises(hb.BackendError):
        hb.InferenceSession(backend, image, addressed=True).close()


def test_two_contexts_at_once():
    """The same calls from two contexts on two streams, interleaved without waiting: each keeps to its own buffers."""
    contexts = []
    for seed in (31, 32):
        be, stream, rng = hb.B200Backend(0), torch.cuda.Stream(), np.random.default_rng(seed)
        be.set_stream(stream.cuda_stream)
        few, many = Cache(rng, [2000, 700], 16, 2, 128, 128), Cache(rng, [1500, 900], 32, 2, 128, 128)
        tensors = [strided(rng, 2, 1024, 1024, "bf16"), strided(rng, 300, 1024, 1024, "bf16"), strided(rng, 300, 256, 256, "bf16"), strided(rng, 300, 256, 256, "bf16")]
        outs = [torch.zeros(n, 1024, dtype=torch.bfloat16, device="cuda") for n in (2, 300, 300)]
        contexts.append((be, few, many, tensors, outs))

    def run(be, few, many, t, outs):
        return [attention(be, few, t[0], None, outs[0], 8, "bf16"), attention(be, many, t[1], [0, 180, 300], outs[1], 8, "bf16"),
                packed(be, t[1], t[2], t[3], [0, 250, 300], outs[2], 8, 2, 128, 128, True, "bf16")]

    wants = []
    for c in contexts:
        kept = run(*c)
        c[0].synchronize()
        wants.append([o.clone() for o in c[4]])
        for o in c[4]:
            o.zero_()
    torch.cuda.synchronize()
    slots = [run(*c) for c in contexts]          # binds once; what follows is only dispatched
    del kept, slots
    for _ in range(10):
        kept = [run(*c) for c in contexts]
    for c in contexts:
        c[0].synchronize()
    for c, want in zip(contexts, wants):
        assert all(torch.equal(a, b) for a, b in zip(c[4], want))
    for c in contexts:
        c[0].close()


@pytest.mark.parametrize("new,lens,block,heads,kv,dim,dtype", [
    ([1] * 3, [3000, 40, 1700], 16, 8, 2, 128, "bf16"),
    ([1] * 2, [3000, 1700], 32, 32, 2, 64, "f16"),
    ([1] * 2, [5000, 1700], 32, 8, 2, 128, "f32"),
    ([200, 90], [3000, 700], 16, 8, 2, 128, "bf16"),
    ([200, 90], [3000, 700], 24, 8, 2, 128, "bf16"),
    ([70, 90], [900, 700], 16, 8, 2, 64, "f32"),
])
def test_block_cache_attention_repeats_its_bits(backend, new, lens, block, heads, kv, dim, dtype):
    """Parts of a sequence are joined in their order, whoever comes last."""
    rng = np.random.default_rng(8)
    cache, rows = Cache(rng, lens, block, kv, dim, dim), sum(new)
    q = strided(rng, rows, heads * dim, heads * dim, dtype)
    outs = [torch.zeros(rows, heads * dim, dtype=TORCH[dtype], device="cuda") for _ in range(6)]
    for o in outs:
        attention(backend, cache, q, starts_of(new), o, heads, dtype)
    backend.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_thousands_of_sequences(backend, dtype):
    """More sequences than any table in shared memory has entries, most of them a token or none."""
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 3, 5000)
    lens[4000] = 150
    starts, rows = starts_of(lens), int(lens.sum())
    q, k, v = (strided(rng, rows, n * 64, n * 64, dtype) for n in (2, 1, 1))
    out = torch.zeros(rows, 128, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, starts, out, 2, 1, 64, 64, True, dtype)
    want, off = packed_reference(q, k, v, starts, 2, 1, 64, 64, True, dtype)
    backend.synchronize()
    check(f64(out), want, off)
    # the same rows over a cache in which each sequence has up to 40 positions
    have = [int(n) + int(rng.integers(0, 38)) if n else 0 for n in lens]
    cache = Cache(rng, have, 16, 1, 64, 64)
    out.zero_()
    attention(backend, cache, q, starts, out, 2, dtype)
    backend.synchronize()
    got, qf = f64(out).reshape(rows, 2, 64), f64(q).reshape(rows, 2, 64)
    for s in np.concatenate([rng.integers(0, 5000, 300), [0, 4000, 4999]]):
        if lens[s]:
            a, m, n = int(starts[s]), int(lens[s]), have[s]
            kh, vh = cache.held("k", s, n)[:, 0], cache.held("v", s, n)[:, 0]
            for h in range(2):
                w, o = attend(qf[a:a + m, h], kh, vh, n - m + 1 + np.arange(m), 0.125, dtype, CACHE_WEIGHT_HALF[dtype])
                check(got[a:a + m, h], w, o, f"sequence {s}")


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [128, 256])
def test_a_cache_of_more_than_32_bits_of_bytes(backend, new, dim):
    """The table names blocks on both sides of 2^31 and 2^32 bytes; the rest of the cache is never touched."""
    rng = np.random.default_rng(10)
    block, vdim = 1024, 16
    blocks = 2 ** 32 // (block * dim) + 40
    k_codes, v_codes = torch.empty(blocks, 1, block, dim, dtype=torch.int8, device="cuda"), torch.empty(blocks, 1, block, vdim, dtype=torch.int8, device="cuda")
    scales = [torch.zeros(blocks, 1, device="cuda") for _ in range(2)]
    named = [blocks - 1, 0, 2 ** 31 // (block * dim), 2 ** 32 // (block * dim)]
    table = i32([named])
    n = 3 * block + 77
    k, v = strided(rng, n, dim, dim, "bf16"), strided(rng, n, vdim, vdim, "bf16")
    s = Slots(backend)
    planes = lambda starts, length: [s(i32(starts)), s(i32([length])), s(table), s(k_codes), s(scales[0]), s(v_codes), s(scales[1])]
    backend.dispatch(kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(s(k), s(v), *planes([0, n], n), n, 1, 1, dim, vdim, dim, vdim, block, blocks, 4, kc.DTYPE_BF16)), s.ws)
    s = Slots(backend)
    q, out = strided(rng, new, 2 * dim, 2 * dim, "bf16"), torch.zeros(new, 2 * vdim, dtype=torch.bfloat16, device="cuda")
    backend.dispatch(kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(s(q), *planes([0, new], n), s(out), new, 1, 2, 1, dim, vdim, 2 * dim, 2 * vdim, block, blocks, 4, 0, kc.DTYPE_BF16)),
                     s.ws)
    backend.synchronize()
    host = {"k": np.zeros((4, 1, block, dim), dtype=np.int8), "v": np.zeros((4, 1, block, vdim), dtype=np.int8)}
    held = {}
    for p, x, codes, scale in (("k", k, k_codes, scales[0]), ("v", v, v_codes, scales[1])):
        want_scales = np.zeros((4, 1), dtype=np.float32)
        write_plane(f64(x).reshape(n, 1, -1), host[p], want_scales, [0, n], [n], np.arange(4)[None], block)
        at = torch.tensor(named, device="cuda")
        assert np.array_equal(scale[at].cpu().numpy(), want_scales)
        got = codes[at].cpu().numpy().reshape(4 * block, -1)[:n]
        assert np.array_equal(got, host[p].reshape(4 * block, -1)[:n])
        held[p] = got.astype(np.float64) * np.repeat(want_scales[:, 0].astype(np.float64), block)[:n, None]
    got, qf = f64(out).reshape(new, 2, vdim), f64(q).reshape(new, 2, dim)
    for h in range(2):
        want, off = attend(qf[:, h], held["k"], held["v"], n - new + 1 + np.arange(new), dim ** -0.5, "bf16", CACHE_WEIGHT_HALF["bf16"])
        check(got[:, h], want, off, f"head {h}")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_packed_rows_of_a_pitch_beyond_32_bits(backend, dtype):
    """300 rows whose offsets pass 2^31 elements, k and v beside q in the same rows."""
    rng = np.random.default_rng(13)
    rows, pitch = 300, 8 * 10 ** 6
    wide = torch.empty(rows * pitch, dtype=TORCH[dtype], device="cuda").view(rows, pitch)
    wide[:, :256] = strided(rng, rows, 256, 256, dtype)
    q, k, v = wide[:, :128], wide[:, 128:192], wide[:, 192:256]
    out = torch.zeros(rows, 128, dtype=TORCH[dtype], device="cuda")
    packed(backend, q, k, v, [0, 90, 300], out, 2, 1, 64, 64, True, dtype)
    backend.synchronize()
    want, off = packed_reference(q, k, v, [0, 90, 300], 2, 1, 64, 64, True, dtype)
    check(f64(out), want, off)
    del wide
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 60])
def test_block_scales_far_apart_and_zero(backend, dtype, new):
    """Value scales from 1 down to 2^-18 of the largest and none at all, key scales of zero; a block of each, and no block with a scale."""
    rng = np.random.default_rng(14)
    cache = Cache(rng, [16 * 19, 16 * 4, 80], 16, 1, 64, 64)
    for j in range(19):
        cache.host["v_scales"][cache.table[0, j]] = np.float32(2.0 ** -j / 127) if j % 5 else 0.0
        cache.host["k_scales"][cache.table[0, j]] = 0.0 if j % 7 == 3 else np.float32(0.01)
    for j in range(4):
        cache.host["v_scales"][cache.table[1, j]] = 0.0
    cache.dev = {n: torch.from_numpy(a.copy()).cuda() for n, a in cache.host.items()}
    rows, starts = 3 * new, np.arange(4) * new
    q, out = strided(rng, rows, 128, 128, dtype), torch.full((rows, 128), 7.0, dtype=TORCH[dtype], device="cuda")
    attention(backend, cache, q, starts, out, 2, dtype)
    backend.synchronize()
    got, qf = f64(out).reshape(rows, 2, 64), f64(q).reshape(rows, 2, 64)
    for s, n in enumerate(cache.lens):
        k, v = cache.held("k", s, n)[:, 0], cache.held("v", s, n)[:, 0]
        for h in range(2):
            a = s * new
            want, off = attend(qf[a:a + new, h], k, v, n - new + 1 + np.arange(new), 0.125, dtype, CACHE_WEIGHT_HALF[dtype])
            check(got[a:a + new, h], want, off, f"sequence {s}")
