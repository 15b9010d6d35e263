"""The operators of a serving step over a paged 8-bit KV cache, as measurable cases.

* ``tables``  one step of the block tables: rows that end give their pages back, rows that grow
              take pages, and every new token gets its slot (``BlockTables.step``);
* ``append``  new keys and values quantized into their slots, then read back from the units they
              went to (``PagedKVCache.append`` and ``.read``);
* ``attend``  attention of one token or of a prompt per sequence (``PagedKVCache.attend``);
* ``sample``  token ids drawn from logits with temperature, top-k, top-p and min-p
              (``sample_tokens``).

The cache holds INT8 codes in pages of ``block`` tokens, each cut into units of 16 tokens that
share one fp32 scale per kv head for the keys and one for the values:
  k_codes [layers, pages, kv_heads, block / 16, 16, D]    k_scales [layers, pages, kv_heads, block / 16]
  v_codes [layers, pages, kv_heads, block / 16, D, 16]    v_scales (the same)

Head counts are those of Llama-3.2-3B (24 / 8), Qwen2.5-7B (28 / 4) and Qwen2.5-14B (40 / 8).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = 16
HEADS = ((24, 8), (28, 4), (40, 8))


def listed():
    return [
        # one decoding step's bookkeeping of a full serving batch: a token each, a page now and then
        dict(name="tables_decode", kind="tables", rows=64, width=2048, block=64, new_low=1, new_high=1,
             finished=0.0, start=700),
        # a burst of admissions: most rows end and take a new prompt in the same step
        dict(name="tables_admit", kind="tables", rows=256, width=256, block=16, new_low=1, new_high=900,
             finished=1.0, start=300),
        # one decoding step's keys and values of a serving batch, mid-page
        dict(name="append_decode", kind="append", rows=64, tokens=1, start=333, kv_heads=8, dim=128, block=64,
             dtype="bf16"),
        # a batch of prompts going into the cache, the first units already begun
        dict(name="append_prompt", kind="append", rows=4, tokens=2048, start=5, kv_heads=8, dim=128, block=64,
             dtype="bf16"),
        # a single user's next token after a short chat prompt: latency
        dict(name="decode_one", kind="attend", rows=1, q_heads=24, kv_heads=8, dim=128, block=64, dtype="bf16",
             low=613, high=613, new=1),
        # a ragged decoding batch on small pages
        dict(name="decode_batch", kind="attend", rows=32, q_heads=28, kv_heads=4, dim=128, block=16, dtype="fp16",
             low=65, high=4099, new=1),
        # long documents: the cache is all there is to read
        dict(name="decode_long", kind="attend", rows=4, q_heads=40, kv_heads=8, dim=128, block=64, dtype="bf16",
             low=131072, high=131072, new=1),
        # a chunk of a long prompt over what came before it
        dict(name="prompt_chunk", kind="attend", rows=1, q_heads=24, kv_heads=8, dim=128, block=64, dtype="bf16",
             low=16384, high=16384, new=512),
        # a batch of whole prompts of unequal lengths
        dict(name="prompt_batch", kind="attend", rows=4, q_heads=24, kv_heads=8, dim=128, block=32, dtype="bf16",
             low=1500, high=2048, new=0),
        # a single user's next token with the usual chat settings
        dict(name="sample_one", kind="sample", rows=1, vocab=128256, dtype="bf16", temperature=0.7, top_k=50,
             top_p=0.9, min_p=0.0, peak=8.0, mixed=False),
        # a batch drawn from the nucleus alone
        dict(name="sample_nucleus", kind="sample", rows=64, vocab=128256, dtype="bf16", temperature=1.0, top_k=0,
             top_p=0.95, min_p=0.0, peak=8.0, mixed=False),
        # a full batch, every request with settings of its own, fp32 logits
        dict(name="sample_mixed", kind="sample", rows=256, vocab=128256, dtype="fp32", temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.05, peak=8.0, mixed=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("tables", "append", "attend", "attend", "sample", "sample"))
    block = rng.choice((16, 32, 64, 128))
    if kind == "tables":
        rows, finished = _log(rng, 1, 512), rng.choice((0.0, 1.0))
        # rows that go on grow by a token at every pass and need a table they never outgrow
        if finished:
            return dict(kind=kind, rows=rows, width=1024 // block * 8, block=block, new_low=0,
                        new_high=_log(rng, 1, max(1, min(800, 200000 // rows))), finished=1.0, start=_log(rng, 1, 4000))
        return dict(kind=kind, rows=min(rows, 128), width=131072 // block, block=block, new_low=0, new_high=1,
                    finished=0.0, start=_log(rng, 1, 4000))
    dim = rng.choice((64, 128, 128))
    if kind == "append":
        rows, tokens = _log(rng, 1, 128), _log(rng, 1, 4096)
        rows = max(1, min(rows, 8192 // tokens))
        return dict(kind=kind, rows=rows, tokens=tokens, start=rng.randrange(0, 200), kv_heads=rng.choice((1, 2, 4, 8)),
                    dim=dim, block=block, dtype=rng.choice(("bf16", "fp16")))
    if kind == "attend":
        q_heads, kv_heads = rng.choice(HEADS + ((8, 8), (16, 1), (32, 8)))
        case = dict(kind=kind, q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=block,
                    dtype=rng.choice(("bf16", "fp16")))
        if rng.random() < 0.6:   # one token, or a few that were guessed ahead
            rows = _log(rng, 1, 128)
            high = max(1, min(_log(rng, 16, 65536), 2 ** 21 // (rows * kv_heads)))
            new = min(high, rng.choice((1, 1, 1, 1, 2, 4)))
            return dict(case, rows=rows, low=max(new, high // rng.choice((1, 2, 8))), high=high, new=new)
        rows = _log(rng, 1, 8)
        high = max(8, min(_log(rng, 64, 8192), 8192 // rows))
        new = rng.choice((0, 0, _log(rng, 8, high)))
        while rows * high * (new or high // 2) * q_heads * dim > 2 * 10 ** 10:
            high, new = max(8, high // 2), min(new, max(8, high // 2))
        return dict(case, rows=rows, low=max(new, high // rng.choice((1, 2, 4)), 1), high=high, new=new)
    return dict(kind=kind, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 128256),
                dtype=rng.choice(("bf16", "fp16", "fp32")), temperature=rng.choice((0.0, 0.6, 0.8, 1.0, 1.3)),
                top_k=rng.choice((0, 1, 20, 50, 400)), top_p=rng.choice((1.0, 0.95, 0.8, 0.5)),
                min_p=rng.choice((0.0, 0.0, 0.02, 0.1)), peak=rng.uniform(2.0, 12.0), mixed=rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------


def _gen(seed, device=DEV):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _ceil(a, b):
    return -(-a // b)


def _lengths(case):
    """Cached tokens of each sequence, the queried ones among them: log-uniform from low to high, the first the longest.
    They go by the case, so that other inputs have the same shapes."""
    low, high, rows = case["low"], case["high"], case["rows"]
    u = torch.rand((rows,), generator=_gen(low + high, "cpu"), dtype=torch.float64)
    n = torch.exp(math.log(low) + u * (math.log(high) - math.log(low))).round().to(torch.int64).clamp(low, high)
    n[0] = high
    return n


def _fill_codes(t, g):
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        part = flat[i:i + (1 << 26)]
        part.copy_(torch.randn((part.numel(),), generator=g, device=DEV).mul_(38.0).round_().clamp_(-127, 127))


def _storage(pages, kv_heads, block, dim, g, filled):
    units = block // UNIT
    k = torch.empty((1, pages, kv_heads, units, UNIT, dim), dtype=torch.int8, device=DEV)
    v = torch.empty((1, pages, kv_heads, units, dim, UNIT), dtype=torch.int8, device=DEV)
    ks = torch.empty((1, pages, kv_heads, units), dtype=torch.float32, device=DEV)
    vs = torch.empty_like(ks)
    if filled:
        _fill_codes(k, g)
        _fill_codes(v, g)
        # absmax / 127 of 16 tokens of unit-variance heads, some heads and places louder than others
        ks.copy_(torch.randn(ks.shape, generator=g, device=DEV).mul_(0.3).exp_().mul_(0.03))
        vs.copy_(torch.randn(vs.shape, generator=g, device=DEV).mul_(0.3).exp_().mul_(0.025))
    else:
        for t in (k, v, ks, vs):
            t.zero_()
    return k, v, ks, vs


def _prepare_tables(case, seed):
    g = _gen(seed, "cpu")
    rows, width, block = case["rows"], case["width"], case["block"]
    start = torch.randint(max(1, case["start"] // 2), case["start"] + 1, (rows,), generator=g)
    new = torch.randint(case["new_low"], case["new_high"] + 1, (rows,), generator=g)
    fin = torch.rand((rows,), generator=g) < case["finished"]
    pages = rows * width
    order = torch.randperm(pages, generator=g).to(torch.int32)
    have = (start + block - 1) // block
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for b in range(rows):
        table[b, :have[b]] = order[at:at + int(have[b])]
        at += int(have[b])
    free = torch.cat([order[at:], torch.full((at,), -1, dtype=torch.int32)])
    return dict(case=case, table=table.to(DEV), lengths=start.to(torch.int32).to(DEV), free=free.to(DEV),
                free_count=torch.tensor([pages - at], dtype=torch.int32, device=DEV), new=new.to(torch.int32).to(DEV),
                finished=fin.to(DEV) if case["finished"] else None, max_tokens=max(1, rows * case["new_high"]))


def _prepare_append(case, seed):
    g, gc = _gen(seed), _gen(seed, "cpu")
    rows, n, block, hkv, dim = case["rows"], case["tokens"], case["block"], case["kv_heads"], case["dim"]
    start = torch.randint(case["start"] // 2, case["start"] + 1, (rows,), generator=_gen(n, "cpu"))
    per = _ceil(case["start"] + n, block)
    pages = rows * per + 3
    table = torch.randperm(pages, generator=gc)[:rows * per].view(rows, per)
    pos = start[:, None] + torch.arange(n)[None, :]
    slots = (table.gather(1, pos // block) * block + pos % block).view(-1)
    unit = slots // UNIT
    first = torch.ones_like(unit, dtype=torch.bool)
    first[1:] = unit[1:] != unit[:-1]
    first.view(rows, n)[:, 0] = True
    units = unit[first]                                       # units in the order they are met
    which = first.cumsum(0) - 1                               # each token's unit
    token_of = torch.full((units.numel(), UNIT), slots.numel())
    token_of[which, slots % UNIT] = torch.arange(slots.numel())
    begun = (slots % UNIT)[first]                             # tokens each unit held before
    # the slots of these units that hold a token afterwards: decoding reads the whole unit back
    lane = torch.arange(UNIT)[None, :]
    live = (token_of < slots.numel()) | (lane < begun[:, None])
    back = torch.where(live, units[:, None] * UNIT + lane, -1).view(-1)
    k, v, ks, vs = _storage(pages, hkv, block, dim, g, True)
    shape = (rows * n, hkv, dim)
    loud = torch.randn((1, hkv, dim), generator=g, device=DEV).mul_(0.5).exp_()
    dt = DTYPES[case["dtype"]]
    return dict(case=case, k=k, v=v, ks=ks, vs=vs, new_k=(torch.randn(shape, generator=g, device=DEV) * loud).to(dt),
                new_v=torch.randn(shape, generator=g, device=DEV).to(dt), slots=slots.to(torch.int32).to(DEV),
                back=back.to(torch.int32).to(DEV), units=units.to(DEV), token_of=token_of.to(DEV),
                begun=begun.to(DEV))


def _prepare_attend(case, seed):
    g, gc = _gen(seed), _gen(seed, "cpu")
    rows, block, dim, hq, hkv = case["rows"], case["block"], case["dim"], case["q_heads"], case["kv_heads"]
    lengths = _lengths(case)
    new = lengths.clone() if case["new"] == 0 else torch.full_like(lengths, case["new"])
    width = _ceil(case["high"], block)
    count = (lengths + block - 1) // block
    pages = int(count.sum())
    order = torch.randperm(pages, generator=gc).to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for b in range(rows):
        table[b, :count[b]] = order[at:at + int(count[b])]
        at += int(count[b])
    k, v, ks, vs = _storage(pages, hkv, block, dim, g, True)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
    q = torch.randn((int(starts[-1]), hq, dim), generator=g, device=DEV).mul_(1.5).to(DTYPES[case["dtype"]])
    return dict(case=case, k=k, v=v, ks=ks, vs=vs, table=table.to(DEV), lengths=lengths.to(torch.int32).to(DEV),
                starts=starts.to(torch.int32).to(DEV), max_new=int(new.max()), q=q, scale=dim ** -0.5,
                row_of=torch.repeat_interleave(torch.arange(rows), new).to(DEV))


def _prepare_sample(case, seed):
    g, gc = _gen(seed), _gen(seed, "cpu")
    rows, vocab = case["rows"], case["vocab"]
    # a bulk of unlikely tokens and a few dozen that the model considers, as next-token logits have
    z = torch.randn((rows, vocab), generator=g, device=DEV).mul_(2.2)
    few = max(2, min(60, vocab // 4))
    at = torch.randint(0, vocab, (rows, few), generator=g, device=DEV)
    z.scatter_(1, at, torch.randn((rows, few), generator=g, device=DEV).mul_(2.5).add_(case["peak"]))
    s = dict(case=case, logits=z.to(DTYPES[case["dtype"]]),
             uniform=torch.rand((rows,), generator=g, device=DEV))
    t, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
    if case["mixed"]:   # every other choice of request parameters, row by row
        pick = lambda xs, dt: torch.tensor(xs, dtype=dt)[torch.randint(0, len(xs), (rows,), generator=gc)].to(DEV)  # noqa: E731
        s.update(t=pick((0.0, 0.5, 0.8, t, 1.2), torch.float32), k=pick((0, 0, 1, 40, 200), torch.int32),
                 p=pick((1.0, 0.95, p, 0.6), torch.float32), m=pick((0.0, 0.0, m, 0.1), torch.float32))
    else:
        full = lambda x, dt: torch.full((rows,), x, dtype=dt, device=DEV)  # noqa: E731
        s.update(t=full(t, torch.float32), k=full(k, torch.int32), p=full(p, torch.float32), m=full(m, torch.float32))
    return s


def prepare(case, seed):
    return {"tables": _prepare_tables, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["kind"]](case, seed)


# ---- the framework's calls ---------------------------------------------------


def _cache(s):
    if "cache" not in s:   # the handle that a program keeps for its cache
        from tilequant_amd.paged_cache import PagedKVCache

        s["cache"] = PagedKVCache(s["k"], s["v"], s["ks"], s["vs"])
    return s["cache"]


def _own_tables(s):
    if "tables" not in s:
        from tilequant_amd.paged_cache import BlockTables

        s["tables"] = BlockTables(s["table"], s["lengths"], s["free"], s["free_count"], s["case"]["block"])
    step = s["tables"].step(s["new"], max_tokens=s["max_tokens"], finished=s["finished"])
    return (step.slots, step.positions, step.query_start, step.granted, s["lengths"], s["table"], s["free_count"])


def _own_append(s):
    cache = _cache(s)
    cache.append(0, s["new_k"], s["new_v"], s["slots"])
    k, v = cache.read(0, s["back"], s["new_k"].dtype)
    return k, v, s["ks"], s["vs"]


def _own_attend(s):
    if s["max_new"] == 1:
        return _cache(s).attend(0, s["q"], s["table"], s["lengths"], scale=s["scale"])
    return _cache(s).attend(0, s["q"], s["table"], s["lengths"], scale=s["scale"], query_start=s["starts"],
                            max_query=s["max_new"])


def _own_sample(s):
    from tilequant_amd.sampling import sample_tokens

    return sample_tokens(s["logits"], s["uniform"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])


# ---- the plain forms ----------------------------------------------------------


def _plain_tables(s):
    table, lengths, free, count, block = s["table"], s["lengths"], s["free"], s["free_count"], s["case"]["block"]
    rows, width = table.shape
    col = torch.arange(width, device=DEV)[None, :]
    cnt = count.long()
    if s["finished"] is not None:
        held = torch.where(s["finished"], (lengths.long() + block - 1) // block, 0)
        before = held.cumsum(0) - held
        gone = col < held[:, None]
        at = torch.where(gone, cnt + before[:, None] + col, free.numel())
        pool = torch.cat([free, free.new_zeros(1)])
        pool[at.view(-1)] = table.view(-1)
        free.copy_(pool[:-1])
        table.copy_(torch.where(gone, -1, table))
        lengths.copy_(torch.where(s["finished"], 0, lengths))
        cnt = cnt + held.sum()
    old = lengths.long()
    n = s["new"].long().clamp(min=0)
    have = (old + block - 1) // block
    fits = old + n <= width * block
    need = torch.where(fits, (old + n + block - 1) // block - have, 0)
    asked = torch.where(fits, n, 0)
    ok = fits & ((need.cumsum(0) <= cnt) | (need == 0)) & (asked.cumsum(0) <= s["max_tokens"])
    need, n = torch.where(ok, need, 0), torch.where(ok, n, 0)
    before = need.cumsum(0) - need
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (cnt - 1 - before[:, None] - (col - have[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[at], table))
    count.copy_((cnt - need.sum()).to(torch.int32))
    lengths.copy_((old + n).to(torch.int32))
    starts = torch.cat([n.new_zeros(1), n.cumsum(0)])
    t = torch.arange(s["max_tokens"], device=DEV)
    row = torch.searchsorted(starts[1:], t, right=True).clamp(max=rows - 1)
    live = t < starts[-1]
    pos = torch.where(live, old[row] + t - starts[row], 0)
    slots = torch.where(live, table[row, (pos // block).clamp(max=width - 1)].long() * block + pos % block, -1)
    return (slots.to(torch.int32), pos.to(torch.int32), starts.to(torch.int32), ok, lengths, table, count)


def _plain_quantize(x, codes, scales, s, transposed):
    """Codes and scales of the touched units after the append; codes [units, heads, 16, D]."""
    x = torch.nan_to_num(x, nan=0.0).float()
    x = torch.cat([x, x.new_zeros((1,) + x.shape[1:])])[s["token_of"]]      # [U, 16, H, D]
    x = x.permute(0, 2, 1, 3)
    per = codes.shape[3]
    page, unit = s["units"] // per, s["units"] % per
    old = codes[0, page, :, unit]                                           # [U, H, 16, D] or [U, H, D, 16]
    old = (old.transpose(2, 3) if transposed else old).float()
    before = torch.where(s["begun"][:, None] > 0, scales[0, page, :, unit], 0.0)
    top = x.abs().amax(dim=(2, 3))
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    after = torch.maximum(before, top / 127.0)
    some = after > 0
    inv = torch.where(some, 1.0 / after, 0.0)[..., None, None]
    fresh = (x * inv).round().clamp(-127, 127)
    kept = (old * torch.where(some, before / after, 0.0)[..., None, None]).round()
    new = torch.where((s["token_of"] < s["slots"].numel())[:, None, :, None], fresh, kept)
    codes[0, page, :, unit] = (new.transpose(2, 3) if transposed else new).to(torch.int8)
    scales[0, page, :, unit] = after


def _plain_read(codes, scales, slots, dtype, transposed):
    per = codes.shape[3]
    at = slots.long().clamp(min=0)
    unit, lane = at // UNIT, at % UNIT
    page, unit = unit // per, unit % per
    c = codes[0, page, :, unit, :, lane] if transposed else codes[0, page, :, unit, lane]   # [N, H, D]
    x = c.float() * scales[0, page, :, unit][..., None]
    return torch.where((slots >= 0)[:, None, None], x, 0.0).to(dtype)


def _plain_append(s):
    _plain_quantize(s["new_k"], s["k"], s["ks"], s, False)
    _plain_quantize(s["new_v"], s["v"], s["vs"], s, True)
    dt = s["new_k"].dtype
    return (_plain_read(s["k"], s["ks"], s["back"], dt, False), _plain_read(s["v"], s["vs"], s["back"], dt, True),
            s["ks"], s["vs"])


def _plain_attend(s):
    case = s["case"]
    rows, dim, hq, hkv = case["rows"], case["dim"], case["q_heads"], case["kv_heads"]
    group, most = hq // hkv, s["max_new"]
    page = s["table"].long().clamp(min=0)                                   # [rows, width]
    k = s["k"][0][page].float() * s["ks"][0][page][..., None, None]          # [rows, width, H, units, 16, D]
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(rows, hkv, -1, dim)
    v = s["v"][0][page].float() * s["vs"][0][page][..., None, None]          # [rows, width, H, units, D, 16]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(rows, hkv, -1, dim)
    starts = s["starts"].long()
    i = torch.arange(most, device=DEV)
    new = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)     # [rows, most]
    q = s["q"][at].float().view(rows, most, hkv, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(rows, hkv, group * most, dim) * s["scale"]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(rows, hkv, group, most, -1)
    last = (s["lengths"].long() - new)[:, None] + i[None, :]                # the last key each query sees
    seen = torch.arange(k.shape[2], device=DEV)[None, None, :] <= last[:, :, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True))
    out = torch.matmul((p / p.sum(dim=-1, keepdim=True)).view(rows, hkv, group * most, -1), v)
    out = out.view(rows, hkv, group, most, dim).permute(0, 3, 1, 2, 4).reshape(rows, most, hq, dim)
    t = torch.arange(s["q"].shape[0], device=DEV)
    return out[s["row_of"], t - starts[s["row_of"]]].to(s["q"].dtype)


def _plain_sample(s):
    z, index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    vocab = z.shape[1]
    z, t = z.double(), s["t"].double()[:, None]                             # sums over the vocabulary: 64 bits
    w = torch.exp((z - z[:, :1]) / torch.where(t > 0, t, 1.0))
    i = torch.arange(vocab, device=DEV)[None, :]
    k = s["k"].long()[:, None]
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    cum = torch.where(i < k, w, 0.0).cumsum(1)
    kept = (i < k) & ((cum - w < s["p"].double()[:, None] * cum[:, -1:]) | (s["p"][:, None] >= 1))
    kept &= w >= s["m"].double()[:, None]
    kept[:, 0] = True
    cum = torch.where(kept, w, 0.0).cumsum(1)
    at = (cum <= s["uniform"].double()[:, None] * cum[:, -1:]).sum(1)
    at = torch.minimum(at, kept.sum(1) - 1)
    at = torch.where(s["t"] > 0, at, 0)
    return index.gather(1, at[:, None])[:, 0]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tables": _own_tables, "append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](state)
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend,
            "sample": _plain_sample}[kind](state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "tables":
        tokens = case["rows"] * (case["new_low"] + case["new_high"]) / 2
        pages = tokens / case["block"] + case["finished"] * case["rows"] * case["start"] * 0.75 / case["block"]
        return {"bytes": 8.0 * tokens + 16.0 * pages + 24.0 * case["rows"] + 8, "flops": 0}
    if kind == "append":
        values = 2.0 * case["rows"] * case["tokens"] * case["kv_heads"] * case["dim"]
        units = case["rows"] * _ceil(case["tokens"] + UNIT // 2, UNIT)
        back = 2.0 * units * UNIT * case["kv_heads"] * case["dim"]
        return {"bytes": values * 3 + back * 3 + 16.0 * units * case["kv_heads"], "flops": values * 2}
    if kind == "attend":
        low, high, rows = case["low"], case["high"], case["rows"]
        mean = high if low == high else (high - low) / math.log(high / low)
        tokens = high + (rows - 1) * mean                    # cached; the first sequence is the longest
        new = tokens if case["new"] == 0 else rows * case["new"]
        row = case["kv_heads"] * (2 * case["dim"] + 8 / UNIT)
        pairs = new * tokens / rows if case["new"] else 0.5 * (high * high + (rows - 1) * (
            high * high if low == high else (high * high - low * low) / (2 * math.log(high / low))))
        if case["new"] > 1:
            pairs -= rows * case["new"] * (case["new"] - 1) / 2
        return {"bytes": tokens * row + 4.0 * new * case["q_heads"] * case["dim"],
                "flops": 4.0 * pairs * case["q_heads"] * case["dim"]}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": float(case["rows"]) * (case["vocab"] * size + 28), "flops": 4.0 * case["rows"] * case["vocab"]}


# ---- the same in 64 bits --------------------------------------------------------


def _exact_append(case, seed):
    s = _prepare_append(case, seed)
    n_tokens = s["slots"].numel()
    got = []
    for x, codes, scales, transposed in ((s["new_k"], s["k"], s["ks"], False), (s["new_v"], s["v"], s["vs"], True)):
        c = codes[0].double()
        c = (c.transpose(-1, -2) if transposed else c).permute(0, 2, 1, 3, 4)          # [pages, units, H, 16, D]
        c = c.reshape(-1, case["kv_heads"], UNIT, case["dim"])[s["units"]]
        flat = scales[0].double().permute(0, 2, 1).reshape(-1, case["kv_heads"]).clone()
        old = flat[s["units"]].masked_fill((s["begun"] == 0)[:, None], 0.0)
        here = s["token_of"] < n_tokens                                                # [U, 16]
        xs = x.double()[s["token_of"].clamp(max=n_tokens - 1)].transpose(1, 2)         # [U, H, 16, D]
        xs = xs.masked_fill(~here[:, None, :, None], 0.0)
        scale = torch.maximum(old, xs.abs().flatten(2).max(dim=2).values / 127)
        new = torch.round(xs / scale[..., None, None])
        c = torch.where(here[:, None, :, None], new, torch.round(c * (old / scale)[..., None, None]))
        flat[s["units"]] = scale
        value = (c * scale[..., None, None]).transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        value = value.masked_fill((s["back"] < 0)[:, None, None], 0.0)
        pages, units = scales.shape[1], scales.shape[3]
        got.append((value, flat.view(1, pages, units, -1).transpose(2, 3).contiguous()))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    hq, hkv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    group = hq // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b in range(case["rows"]):
        n = lengths[b]
        page = s["table"][b, :_ceil(n, case["block"])].long()
        lo, hi = starts[b], starts[b + 1]
        for h in range(hkv):
            k = (s["k"][0, page, h].double() * s["ks"][0, page, h].double()[..., None, None]).reshape(-1, dim)[:n]
            v = s["v"][0, page, h].double() * s["vs"][0, page, h].double()[..., None, None]
            v = v.transpose(-1, -2).reshape(-1, dim)[:n]
            for a in range(lo, hi, 512):
                e = min(hi, a + 512)
                q = s["q"][a:e, h * group:(h + 1) * group].double()                   # [m, group, D]
                score = (q.reshape(-1, dim) @ k.t()).view(e - a, group, n) * s["scale"]
                last = n - (hi - lo) + torch.arange(a - lo, e - lo, device=DEV)
                score.masked_fill_((torch.arange(n, device=DEV)[None, :] > last[:, None])[:, None], -math.inf)
                out[a:e, h * group:(h + 1) * group] = (torch.softmax(score, -1).view(-1, n) @ v).view(e - a, group, dim)
    return out


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    return None   # whole numbers: they are equal or wrong
