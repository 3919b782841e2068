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


def test_no_host_workspace_form(backend):
    host = hb.HostWorkspace([np.zeros(4096, dtype=np.uint8) for _ in range(10)])
    for call in (kc.KernelCall.PackedAttention(kc.PackedAttentionCall()), kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall()),
                 kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall()), kc.KernelCall.LogitRules(kc.LogitRulesCall())):
        with pytest.raises(hb.BackendError, match="no host-workspace form"):
            backend.dispatch(call, host)
