"""The calls of a serving step over several sequences, as far as no GPU is needed: struct layout, wire form, the reference's own arithmetic."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import hologram_b200 as hb
from hologram_b200 import holo
from hologram_b200 import kernel_call as kc
from serving_step_reference import encode, rules, write_plane

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CALLS = {"PackedAttention": kc.PackedAttentionCall, "BlockCacheWrite": kc.BlockCacheWriteCall, "BlockCacheAttention": kc.BlockCacheAttentionCall, "LogitRules": kc.LogitRulesCall}


def test_struct_layout_matches_the_header():
    lines = []
    for name, struct in CALLS.items():
        lines.append(f'printf("%zu\\n", sizeof(Holo{name}Call));')
        lines += [f'printf("%zu\\n", offsetof(Holo{name}Call, {f}));' for f, _ in struct._fields_]
    with tempfile.TemporaryDirectory() as d:
        source, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        with open(source, "w") as f:
            f.write("#include <stdio.h>\n#include <stddef.h>\n#include \"hologram_b200.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), source, "-o", exe])
        got = [int(v) for v in subprocess.check_output([exe]).split()]
    want = []
    for struct in CALLS.values():
        want.append(ctypes.sizeof(struct))
        want += [getattr(struct, f).offset for f, _ in struct._fields_]
    assert got == want


def one_call_archive(name, rows=2):
    """An archive of one call, every operand a port of its own."""
    struct = CALLS[name]
    c = struct()
    w = holo.HoloWriter()
    slot = 0
    for f, kind in struct._fields_:
        if kind is kc.BufferRef:
            setattr(c, f, kc.rb(slot))
            slot += 1
    numbers = dict(rows=rows, sequences=2, heads=4, kv_heads=2, dim=16, vdim=16, q_ld=64, k_ld=32, v_ld=32, ld=64, causal=1, block_rows=16, blocks=3, table_ld=2, vocab=64, out_ld=64,
                   history_ld=4, biases=4, mask_rows=2, mask_ld=2, dtype=kc.DTYPE_F32)
    for f, kind in struct._fields_:
        if kind is not kc.BufferRef and f in numbers:
            setattr(c, f, numbers[f])
    w.calls.append(getattr(kc.KernelCall, name)(c))
    for s in range(slot):
        w.inputs.append(holo.Port(f"p{s}", s, 64, kc.DTYPE_F32, [64]))
    w.exec_plan = [[0]]
    w.slot_bytes = [4096] * slot
    return w.finish()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_archives_hold_the_calls(name):
    assert hb.archive_check(one_call_archive(name))[0] == 1
    with pytest.raises(hb.BackendError):
        hb.archive_check(one_call_archive(name, rows=0))


def test_nearest_codes_in_32_bits():
    """The kernel's estimate and remainder in 32 bits give the code of the exact quotient, ties included."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(40000), rng.integers(-254, 255, 20000) / 2.0, rng.standard_normal(20000) * 1e-30]).astype(np.float32)
    for size in (127.0, 4.0, 1.0, 3.3e38, 1e-30, 254.0):
        scale = np.float32(size) / np.float32(127.0)
        y = x[np.abs(x) <= size]
        inv = np.float32(1.0) / scale
        n = np.rint(y * inv)
        r = (y.astype(np.longdouble) - n.astype(np.longdouble) * np.longdouble(scale)).astype(np.float32)      # fma: one rounding
        odd = (n.astype(np.int64) & 1) != 0
        twice = np.float32(2.0) * r
        n = np.where((twice > scale) | ((twice == scale) & odd), n + 1, np.where((twice < -scale) | ((twice == -scale) & odd), n - 1, n))
        assert np.array_equal(np.clip(n, -127, 127).astype(np.int8), encode(y, scale))


def test_the_status_of_bad_tables_is_no_other_failure_s():
    import re
    folder = os.path.join(ROOT, "hologram_b200", "csrc")
    used, own = set(), None
    for name in os.listdir(folder):
        if name.endswith((".cu", ".cuh", ".h", ".cpp")):
            text = open(os.path.join(folder, name)).read()
            used |= {int(n) for n in re.findall(r"atomicOr\([^;]*?status, (\d+)u\)", text)}
            own = next((int(n) for n in re.findall(r"HOLO_STATUS_TABLE = (\d+)u", text)), own)
    assert {1, 2, 4, 8} <= used and own and not any(own & n for n in used)


def test_division_by_a_product():
    """n // d for n below 2^31 as (n + (m n >> 32)) >> l with 2^l >= d, m = (2^l - d) 2^32 // d + 1, all of 32 bits."""
    rng = np.random.default_rng(3)
    for d in [1, 2, 3, 5, 7, 8, 10, 12, 16, 24, 33, 48, 63, 64, 65, 100, 127, 128, 255, 257, 512, 513, 1000, 1023, 1024, 65535, 2 ** 20 + 1, 2 ** 31 - 1]:
        l = (d - 1).bit_length()
        m = ((2 ** l - d) << 32) // d + 1
        assert m < 2 ** 32
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, 2 ** 31 - 1, 2 ** 31 - 2, (2 ** 31 - 1) // d * d, (2 ** 31 - 1) // d * d - 1] + rng.integers(0, 2 ** 31, 500).tolist():
            if n < 2 ** 31:
                high = m * n >> 32
                assert n + high < 2 ** 32 and (n + high) >> l == n // d


def test_every_touched_block_is_one_item_of_the_write():
    """Sequence s owns items starts[s] / block + 2 s and on; no two sequences share one and none runs out of them."""
    rng = np.random.default_rng(1)
    for _ in range(300):
        block = int(rng.integers(1, 40))
        new = rng.integers(0, 90, rng.integers(1, 12))
        before = rng.integers(0, 200, new.size)
        starts = np.concatenate([[0], np.cumsum(new)])
        seen = set()
        for s, (n, p) in enumerate(zip(new, before)):
            own, after = starts[s] // block + 2 * s, starts[s + 1] // block + 2 * (s + 1)
            touched = (p + n - 1) // block - p // block + 1 if n else 0
            assert touched <= after - own
            for t in range(own, own + touched):
                assert t not in seen and t < starts[-1] // block + 2 * new.size
                seen.add(t)


def test_the_reference_write_keeps_values_within_half_a_step():
    rng = np.random.default_rng(2)
    codes, scales = np.zeros((3, 2, 16, 8), dtype=np.int8), np.zeros((3, 2), dtype=np.float32)
    table, kept = np.array([[2, 0, 1]], dtype=np.int32), []
    for length in range(1, 41):
        x = rng.standard_normal((1, 2, 8)) * rng.choice([0.1, 1.0, 5.0])
        kept.append(x[0])
        write_plane(x, codes, scales, [0, 1], [length], table, 16)
        for p, want in enumerate(kept):
            b = table[0, p // 16]
            # half a step when it was written and half a step of each larger scale: a scale that grows by less than two may do so often
            assert np.all(np.abs(codes[b, :, p % 16] * scales[b][:, None].astype(np.float64) - want) <= 0.5001 * scales[b][:, None] * (1 + min(length - p - 1, 15)))


def test_the_reference_rules():
    z, off = rules(np.array([2.0, -2.0, 1.0, 0.5, 0.0]), [0, 1, 1, 7, -1], (1, 5), (2.0, 0.5, 0.25, 0.5), [(2, 1.0), (2, 3.0), (9, 1.0)], np.array([1, 1, 1, 1, 0], dtype=bool))
    assert z.tolist() == [2.0, (-4.0 - 1.0) * 2, 8.0, 1.0, -np.inf] and np.all(off >= 0)
