"""Operators of a serving step over several sequences: attention of packed prompts, an 8-bit cache in blocks, attention over it, rules on logits.

  packed   attention of whole prompts of different lengths, one behind another (`PackedAttention`)
  write    new key and value rows into a cache of int8 blocks, one scale for each block and head (`BlockCacheWrite`)
  cache    attention of single tokens or portions of several sequences over that cache (`BlockCacheAttention`)
  rules    penalties for repeated tokens, biases, temperature and grammar masks on logits (`LogitRules`)

Where `own` is false `run` computes them with elementary torch operations in 32 bits, padded to the longest sequence; where it is true through
`B200Backend.dispatch`. A cache's codes are whole numbers and come back as such beside their scales: codes * scales are the values held.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # three short prompts that arrive together: the smallest call
        {"name": "packed bf16 8/8x64 1,17,40", "kind": "packed", "dtype": "bf16", "heads": 8, "kv_heads": 8, "dim": 64, "causal": True, "lens": "1,17,40"},
        # a batch of prompts at the decoder's head layout (32 query heads over 8, dim 128), one of them long, one a single token
        {"name": "packed bf16 32/8x128 8192 rows", "kind": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "causal": True,
         "lens": "4096,1337,511,64,1,1953,230"},
        # documents for an encoder, both directions, in one call
        {"name": "packed f16 12/12x64 documents", "kind": "packed", "dtype": "f16", "heads": 12, "kv_heads": 12, "dim": 64, "causal": False,
         "lens": "381,77,512,128,9,256,300,45,510,33,201,190,64,411,350,129"},
        # an f32 model's prompts (the attention benchmark's 12 heads over 2)
        {"name": "packed f32 12/2x128 700,381,55", "kind": "packed", "dtype": "f32", "heads": 12, "kv_heads": 2, "dim": 128, "causal": True, "lens": "700,381,55"},
        # one token of each of 64 decoding sequences at 4096 positions or fewer, most blocks half filled
        {"name": "write bf16 64 tokens", "kind": "write", "dtype": "bf16", "kv_heads": 8, "dim": 128, "block": 32, "lens": ",".join(str(4096 - 37 * i) for i in range(64)),
         "new": ",".join(["1"] * 64)},
        # whole prompts into the cache, one of them behind what an earlier portion left
        {"name": "write bf16 8192 prompt rows", "kind": "write", "dtype": "bf16", "kv_heads": 8, "dim": 128, "block": 32, "lens": "4096,1337,511,64,1,2965,230",
         "new": "4096,1337,511,64,1,1953,230"},
        # a decoding batch at the decoder's widths: 64 sequences, 4096 positions or fewer
        {"name": "cache bf16 32/8x128 b64 4096", "kind": "cache", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 32,
         "lens": ",".join(str(4096 - 37 * (i % 8)) for i in range(64)), "new": ",".join(["1"] * 64)},
        # one sequence with a very long past
        {"name": "cache f16 32/8x128 b1 131000", "kind": "cache", "dtype": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "lens": "131000", "new": "1"},
        # a few short f32 sequences, one of them with nothing cached yet: latency counts
        {"name": "cache f32 12/2x64 b5", "kind": "cache", "dtype": "f32", "heads": 12, "kv_heads": 2, "dim": 64, "block": 16, "lens": "1,333,0,1800,97", "new": "1,1,0,1,1"},
        # portions of four prompts over what their earlier portions left
        {"name": "cache bf16 32/8x128 portions", "kind": "cache", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "lens": "2048,5000,701,8100", "new": "128,256,77,128"},
        # the logits of 64 decoding sequences, all rules in use
        {"name": "rules f32 64x32000", "kind": "rules", "dtype": "f32", "rows": 64, "vocab": 32000, "history": 4096, "bias": 40, "mask": True},
        # one sequence's logits over a large vocabulary: latency counts
        {"name": "rules bf16 1x131072", "kind": "rules", "dtype": "bf16", "rows": 1, "vocab": 131072, "history": 900, "bias": 0, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(t) for t in text.split(",")]


def draw(rng):
    kind = rng.choice(["packed", "packed", "write", "cache", "cache", "rules"])
    heads, kv_heads = rng.choice([(32, 8), (12, 2), (12, 12), (16, 2), (8, 8), (8, 1)])
    if kind == "packed":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        count = rng.randint(1, 8)
        lens = [_log(rng, 1, (3300 if dtype != "f32" else 900) / math.sqrt(count)) for _ in range(count)]
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([48, 64, 80, 128]), "causal": rng.random() < 0.75, "lens": _text(lens)}
    if kind == "rules":
        return {"kind": kind, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "rows": _log(rng, 1, 64), "vocab": _log(rng, 500, 32000), "history": _log(rng, 1, 4096),
                "bias": rng.choice([0, 1, 7, 40]), "mask": rng.random() < 0.6}
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128]), "block": rng.choice([16, 32, 64, 128])}
    if kind == "cache":
        case["heads"] = heads
    if rng.random() < 0.6:      # single tokens
        lens = [_log(rng, 1, 4096) for _ in range(_log(rng, 1, 64))]
        new = [1] * len(lens)
    else:                       # portions
        new = [_log(rng, 1, 256) for _ in range(rng.randint(1, 4))]
        lens = [n + rng.choice([0, _log(rng, 1, 4000)]) for n in new]
    case["lens"], case["new"] = _text(lens), _text(new)
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(gen, rng, lens, block, kv_heads, dim):
    """A cache whose blocks hold what earlier writes left, handed out in no order; some blocks belong to nobody."""
    need = [-(-n // block) for n in lens]
    blocks = sum(need) + 3
    order = list(range(blocks))
    rng.shuffle(order)
    width = max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        for j in range(n):
            table[s, j] = order.pop()
    planes = {}
    for name in ("k", "v"):
        planes[name + "_codes"] = (torch.randn(blocks, kv_heads, block, dim, device="cuda", generator=gen) * 36).round().clamp(-127, 127).to(torch.int8)
        planes[name + "_scales"] = torch.exp(0.2 * torch.randn(blocks, kv_heads, device="cuda", generator=gen)) / 36
    return dict(planes, table=table.cuda())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    rng = random.Random(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    st = {"case": case}
    if case["kind"] == "packed":
        lens = _ints(case["lens"])
        rows = sum(lens)
        st.update(q=normal(rows, case["heads"], case["dim"]), k=normal(rows, case["kv_heads"], case["dim"]), v=normal(rows, case["kv_heads"], case["dim"]),
                  starts=_i32(_starts(lens)), longest=max(lens))
    elif case["kind"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        st["logits"] = (3.0 * torch.randn(rows, vocab, device="cuda", generator=gen)).to(dtype)
        # tokens repeat as text does: few of them make up most of a history
        total = [rng.randint((case["history"] + 1) // 2, case["history"]) for _ in range(rows)]
        st["spans"] = _i32([[rng.randint(0, t), t] for t in total])
        st["history"] = (torch.rand(rows, case["history"], device="cuda", generator=gen) ** 3 * vocab).to(torch.int32)
        st["params"] = torch.tensor([[rng.choice([1.0, 1.1, 1.3]), rng.choice([0.0, 0.5]), rng.choice([0.0, 0.25]), rng.choice([0.0, 0.7, 1.0])] for _ in range(rows)],
                                    device="cuda")
        ids = [sorted(rng.sample(range(vocab), case["bias"])) for _ in range(rows)]
        st["bias_starts"] = _i32(_starts([len(i) for i in ids]))
        st["bias_ids"] = _i32([t for i in ids for t in i])
        st["bias_values"] = 2.0 * torch.randn(rows * case["bias"], device="cuda", generator=gen)
        words = -(-vocab // 32)
        # a grammar's states allow half of the vocabulary; some rows are under no grammar
        st["masks"] = torch.randint(-2 ** 31, 2 ** 31, (4, words), device="cuda", generator=gen, dtype=torch.int64).to(torch.int32) if case["mask"] else None
        st["mask_of"] = _i32([rng.choice([-1, 0, 1, 2, 3]) if rows > 1 else 2 for _ in range(rows)]) if case["mask"] else None
    else:
        lens, new = _ints(case["lens"]), _ints(case["new"])
        st.update(_cache(gen, rng, lens, case["block"], case["kv_heads"], case["dim"]))
        st.update(starts=_i32(_starts(new)), lengths=_i32(lens), longest=max(lens), most=max(new))
        rows = sum(new)
        if case["kind"] == "cache":
            st["q"] = normal(rows, case["heads"], case["dim"])
        else:
            st.update(k=normal(rows, case["kv_heads"], case["dim"]), v=normal(rows, case["kv_heads"], case["dim"]))
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _padded(x, starts, longest):
    """Rows of packed sequences as [sequences, longest, ...] in 32 bits, and which of them are rows of their sequence."""
    at = starts[:-1, None] + torch.arange(longest, device=x.device)
    there = at < starts[1:, None]
    return x[torch.where(there, at, 0)].float(), there


def _attend(q, k, v, seen, scale):
    """q [n, m, heads, dim], k and v [n, keys, kv_heads, dim], seen [n, m, keys] -> [n, m, heads, dim]; rows that see nothing are zero."""
    n, m, heads, dim = q.shape
    kv_heads = k.shape[2]
    q = q.view(n, m, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(n, kv_heads, -1, dim), k.permute(0, 2, 3, 1)).view(n, kv_heads, heads // kv_heads, m, -1)
    s = (s * scale).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    o = torch.matmul(e.view(n, kv_heads, -1, e.shape[-1]), v.permute(0, 2, 1, 3)).view(n, kv_heads, heads // kv_heads, m, -1)
    o = o / e.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(n, m, heads, -1)


def _plain_packed(st):
    case, starts, longest = st["case"], st["starts"].long(), st["longest"]
    q, there = _padded(st["q"], starts, longest)
    k, _ = _padded(st["k"], starts, longest)
    v, _ = _padded(st["v"], starts, longest)
    at = torch.arange(longest, device=q.device)
    seen = there[:, None, :] & (at[:, None] >= at[None, :]) if case["causal"] else there[:, None, :].expand(-1, longest, -1)
    return _attend(q, k, v, seen, case["dim"] ** -0.5)[there].to(st["q"].dtype)


def _held(codes, scales, table):
    """The values of the blocks of `table` as [sequences, positions, kv_heads, dim]."""
    at = table.long().clamp_min(0)
    x = codes[at].float() * scales[at][..., None, None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_cache(st):
    case, starts, lengths = st["case"], st["starts"].long(), st["lengths"].long()
    q, there = _padded(st["q"], starts, st["most"])
    k, v = (_held(st[p + "_codes"], st[p + "_scales"], st["table"]) for p in "kv")
    i = torch.arange(st["most"], device=q.device)
    limit = (lengths - (starts[1:] - starts[:-1]))[:, None] + i + 1
    seen = torch.arange(k.shape[1], device=q.device) < limit[:, :, None]
    return _attend(q, k, v, seen, case["dim"] ** -0.5)[there].to(st["q"].dtype)


def _nearest(x, scale):
    """Codes of x (64 bits) under `scale`: a quotient next to a half needs more than 32 bits."""
    return torch.where(scale > 0, torch.round(x / scale.double().clamp_min(1e-300)), 0.0).clamp(-127, 127).to(torch.int8)


def _plain_write_plane(x, codes, scales, st):
    block, starts, lengths = st["case"]["block"], st["starts"].long(), st["lengths"].long()
    first = lengths - (starts[1:] - starts[:-1])            # a sequence's first new position
    row = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = first[seq] + row - starts[seq]
    home = st["table"][seq, pos // block].long()
    x, full = x.float(), torch.full_like(scales, 127.0)     # a tensor: a quotient by a number is a product with its reciprocal
    most = torch.zeros_like(scales).index_reduce_(0, home, x.abs().amax(-1), "amax") / full
    # the block that held tokens before: its scale only grows, and what it holds is said in the new one
    part = st["table"].gather(1, (first // block).clamp_max(st["table"].shape[1] - 1)[:, None])[:, 0].long()
    half = (first % block != 0) & (starts[1:] > starts[:-1])
    before = scales[part.clamp_min(0)]
    scales[home] = most[home]
    grown = torch.where(half[:, None], torch.maximum(before, most[part.clamp_min(0)]), 0.0)
    part, grown, before, count = part[half], grown[half], before[half], (first % block)[half]
    scales[part] = grown
    old = codes[part]
    again = _nearest(old.double() * before.double()[..., None, None], grown[..., None, None])
    codes[part] = torch.where((torch.arange(block, device=x.device) < count[:, None])[:, None, :, None], again, old)
    codes[home, :, pos % block] = _nearest(x.double(), scales[home][..., None])


def _plain_write(st):
    _plain_write_plane(st["k"], st["k_codes"], st["k_scales"], st)
    _plain_write_plane(st["v"], st["v_codes"], st["v_scales"], st)
    return {p: st[p] for p in ("k_codes", "k_scales", "v_codes", "v_scales")}


def _plain_rules(st):
    z, spans, history = st["logits"].float(), st["spans"].long(), st["history"].long()
    rows, vocab = z.shape
    at = torch.arange(history.shape[1], device=z.device)
    seen = torch.zeros_like(z).scatter_add_(1, history, (at < spans[:, 1:]).float())
    made = torch.zeros_like(z).scatter_add_(1, history, ((at >= spans[:, :1]) & (at < spans[:, 1:])).float())
    again, presence, frequency, temperature = (p[:, None] for p in st["params"].unbind(1))
    z = torch.where(seen > 0, torch.where(z > 0, z / again, z * again), z)
    z = z - (frequency * made + presence * (made > 0))
    entry = torch.arange(st["bias_ids"].numel(), device=z.device)
    z[torch.searchsorted(st["bias_starts"].long(), entry, right=True) - 1, st["bias_ids"].long()] += st["bias_values"]
    z = z / torch.where(temperature > 0, temperature, 1.0)
    if st["masks"] is not None:
        token = torch.arange(vocab, device=z.device)
        allowed = (st["masks"][:, token // 32] >> (token % 32).int()) & 1
        z = z.masked_fill((st["mask_of"] >= 0)[:, None] & (allowed[st["mask_of"].long().clamp_min(0)] == 0), -math.inf)
    return z.to(st["logits"].dtype)


# ---- the framework's calls ---------------------------------------------------------------------------------------------

_kept = {}


def _backend():
    import hologram_b200 as hb
    if "backend" not in _kept:
        _kept["backend"] = hb.B200Backend(torch.cuda.current_device())
    stream = torch.cuda.current_stream().cuda_stream
    if (_kept["backend"].stream or 0) != stream:
        _kept["backend"].set_stream(stream)
    return _kept["backend"]


def _plan(st):
    """The call, its workspace and its result's buffer, which a program makes once for these buffers."""
    import hologram_b200 as hb
    from hologram_b200 import kernel_call as kc
    case, rb = st["case"], kc.rb
    tag = {"bf16": kc.DTYPE_BF16, "f16": kc.DTYPE_F16, "f32": kc.DTYPE_F32}[case["dtype"]]
    ws = hb.DeviceWorkspace(_backend(), 12)
    slots = []

    def ref(tensor):
        if tensor is None or tensor.numel() == 0:
            return kc.NONE
        slots.append(tensor)
        ws.bind(len(slots) - 1, tensor.data_ptr(), tensor.numel() * tensor.element_size())
        return rb(len(slots) - 1)

    if case["kind"] == "packed":
        h, kv, d, rows = case["heads"], case["kv_heads"], case["dim"], st["q"].shape[0]
        out = torch.zeros_like(st["q"])
        call = kc.KernelCall.PackedAttention(kc.PackedAttentionCall(
            ref(st["q"]), ref(st["k"]), ref(st["v"]), ref(st["starts"]), ref(out), rows, st["starts"].numel() - 1, h, kv, d, d, h * d, kv * d, kv * d, h * d, 0,
            int(case["causal"]), tag))
    elif case["kind"] == "rules":
        rows, vocab = st["logits"].shape
        out = torch.empty_like(st["logits"])
        call = kc.KernelCall.LogitRules(kc.LogitRulesCall(
            ref(st["logits"]), ref(st["history"]), ref(st["spans"]), ref(st["params"]),
            ref(st["bias_starts"] if case["bias"] else None), ref(st["bias_ids"]), ref(st["bias_values"]), ref(st["masks"]),
            ref(st["mask_of"]), ref(out), rows, vocab, vocab, vocab, st["history"].shape[1], st["bias_ids"].numel(), 0 if st["masks"] is None else 4, (vocab + 31) // 32,
            tag))
    else:
        kv, d, n = case["kv_heads"], case["dim"], st["lengths"].numel()
        cache = [st[p] for p in ("starts", "lengths", "table", "k_codes", "k_scales", "v_codes", "v_scales")]
        blocks, width = st["k_codes"].shape[0], st["table"].shape[1]
        if case["kind"] == "write":
            out = {p: st[p] for p in ("k_codes", "k_scales", "v_codes", "v_scales")}
            call = kc.KernelCall.BlockCacheWrite(kc.BlockCacheWriteCall(
                ref(st["k"]), ref(st["v"]), *[ref(t) for t in cache], st["k"].shape[0], n, kv, d, d, kv * d, kv * d, case["block"], blocks, width, tag))
        else:
            h = case["heads"]
            out = torch.zeros_like(st["q"])
            call = kc.KernelCall.BlockCacheAttention(kc.BlockCacheAttentionCall(
                ref(st["q"]), *[ref(t) for t in cache], ref(out), st["q"].shape[0], n, h, kv, d, d, h * d, h * d, case["block"], blocks, width, 0, tag))
    return ws, call, out


def run(st):
    if own:
        if "plan" not in st:
            st["plan"] = _plan(st)
        ws, call, out = st["plan"]
        _backend().dispatch(call, ws)
        return out
    return {"packed": _plain_packed, "write": _plain_write, "cache": _plain_cache, "rules": _plain_rules}[st["case"]["kind"]](st)


def work(case):
    es = BYTES[case["dtype"]]
    if case["kind"] == "rules":
        # a history token is read once, a grammar's words once for each row under it
        return {"bytes": case["rows"] * (2 * es * case["vocab"] + 3 * case["history"] + 8 * case["bias"] + (case["vocab"] // 8 if case["mask"] else 0)), "flops": 6 * case["rows"] * case["vocab"]}
    lens, d = _ints(case["lens"]), case["dim"]
    if case["kind"] == "packed":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * 2 * es * d * (case["heads"] + case["kv_heads"]), "flops": 4 * pairs * case["heads"] * d}
    new, kv = _ints(case["new"]), case["kv_heads"]
    if case["kind"] == "write":
        blocks = sum(-(-n // case["block"]) - (n - m) // case["block"] for n, m in zip(lens, new))
        return {"bytes": 2 * kv * (sum(new) * d * (es + 1) + 4 * blocks), "flops": 4 * sum(new) * kv * d}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
    scales = sum(-(-n // case["block"]) for n in lens)
    return {"bytes": 2 * kv * (sum(lens) * d + 4 * scales) + 2 * es * sum(new) * case["heads"] * d, "flops": 4 * pairs * case["heads"] * d}


# ---- in 64 bits --------------------------------------------------------------------------------------------------------


def _exact_attention(q, k, v, first, causal):
    """Rows q [m, heads, dim] at positions first, first + 1, ... over k and v [keys, kv_heads, dim], a kv head at a time."""
    m, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(m, heads, v.shape[2], dtype=torch.float64, device=q.device)
    if k.shape[0] == 0:
        return out
    hidden = torch.arange(k.shape[0], device=q.device)[None, :] > (first + torch.arange(m, device=q.device))[:, None]
    for h in range(heads):
        s = q[:, h] @ k[:, h // group].T / math.sqrt(dim)
        if causal:
            s[hidden] = -math.inf
        out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "packed":
        q, k, v = (st[n].double() for n in "qkv")
        at = st["starts"].tolist()
        return torch.cat([_exact_attention(q[a:b], k[a:b], v[a:b], 0, case["causal"]) for a, b in zip(at, at[1:])])
    if case["kind"] == "rules":
        z = st["logits"].double().cpu().numpy()
        history, spans, params = st["history"].tolist(), st["spans"].tolist(), st["params"].double().tolist()
        at, ids, values = st["bias_starts"].tolist(), st["bias_ids"].tolist(), st["bias_values"].double().tolist()
        for r in range(z.shape[0]):
            again, presence, frequency, temperature = params[r]
            prompt, total = spans[r]
            for t in set(history[r][:total]):
                z[r, t] = z[r, t] / again if z[r, t] > 0 else z[r, t] * again
            for t in history[r][prompt:total]:
                z[r, t] -= frequency
            for t in set(history[r][prompt:total]):
                z[r, t] -= presence
            for e in range(at[r], at[r + 1]):
                z[r, ids[e]] += values[e]
            if temperature:
                z[r] /= temperature
            if case["mask"] and st["mask_of"][r] >= 0:
                words = st["masks"][st["mask_of"][r]].tolist()
                for t in range(z.shape[1]):
                    if not words[t >> 5] >> (t & 31) & 1:
                        z[r, t] = -math.inf
        return torch.from_numpy(z)
    at, lens, table, block = st["starts"].tolist(), st["lengths"].tolist(), st["table"].tolist(), case["block"]
    if case["kind"] == "cache":
        outs = []
        for s, n in enumerate(lens):
            home = table[s][:-(-n // block)]
            k, v = (torch.cat([st[p + "_codes"][b].double() * st[p + "_scales"][b].double()[:, None, None] for b in home] or [st[p + "_codes"][0].double()[:, :0]], 1)[:, :n].transpose(0, 1)
                    for p in "kv")
            outs.append(_exact_attention(st["q"][at[s]:at[s + 1]].double(), k, v, n - (at[s + 1] - at[s]), True))
        return torch.cat(outs)
    result = {}
    for p in "kv":
        codes, scales, x = st[p + "_codes"].clone(), st[p + "_scales"].clone(), st[p].double()
        for s, n in enumerate(lens):
            first = n - (at[s + 1] - at[s])
            for j in range(first // block, -(-n // block)):
                b, lo, hi = table[s][j], max(first, j * block), min(n, (j + 1) * block)
                rows = x[at[s] + lo - first:at[s] + hi - first].transpose(0, 1)          # [kv_heads, rows, dim]
                scale = (rows.abs().amax((1, 2)) / 127).float()
                if lo > j * block:
                    scale = torch.maximum(scale, scales[b])
                    codes[b, :, :lo - j * block] = torch.round(codes[b, :, :lo - j * block].double() * scales[b].double()[:, None, None] / scale.double()[:, None, None]).to(torch.int8)
                codes[b, :, lo - j * block:hi - j * block] = torch.round(rows / scale.double()[:, None, None]).clamp(-127, 127).to(torch.int8)
                scales[b] = scale
        result[p + "_codes"], result[p + "_scales"] = codes, scales.double()
    return {n: result[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
