"""GPU: block tables, the quantized append, read-back and attention of the paged INT8 cache against plain forms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as ref
from tilequant_amd.paged_cache import BlockTables, PagedKVCache, paged_attention_workspace

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- block tables ---------------------------------------------------------------


class TablesPair:
    """BlockTables beside the plain form."""

    def __init__(self, rows, width, pages, block):
        self.gpu = BlockTables.allocate(requests=rows, blocks_per_request=width, blocks=pages, block_size=block, device=DEV)
        self.table = [[-1] * width for _ in range(rows)]
        self.lengths, self.free, self.count, self.block = [0] * rows, list(range(pages - 1, -1, -1)), pages, block

    def step(self, new, max_tokens, finished=None):
        got = self.gpu.step(i32(new), max_tokens=max_tokens,
                            finished=None if finished is None else torch.tensor(finished, device=DEV))
        slots, pos, starts, granted, self.count = ref.tables_step(self.table, self.lengths, self.free, self.count, new,
                                                                  finished, self.block, max_tokens)
        assert got.slots.tolist() == slots and got.positions.tolist() == pos
        assert got.query_start.tolist() == starts and got.granted.tolist() == granted
        assert self.gpu.lengths.tolist() == self.lengths and self.gpu.free_count.tolist() == [self.count]
        assert self.gpu.block_table.tolist() == self.table
        assert self.gpu.free_blocks.tolist()[:self.count] == self.free[:self.count]
        return got


@pytest.mark.parametrize("rows,width,pages,block,most", [(1, 4, 4, 16, 9), (3, 8, 17, 16, 64), (64, 9, 300, 64, 64),
                                                         (65, 9, 300, 32, 500), (200, 40, 3000, 16, 5000),
                                                         (1500, 6, 4000, 16, 3000), (2100, 3, 3000, 1, 4500)])
def test_tables_follow_the_plain_form(rows, width, pages, block, most):
    g = torch.Generator().manual_seed(rows)
    t = TablesPair(rows, width, pages, block)
    per = max(1, most // rows)
    draw = lambda lo, hi: torch.randint(lo, hi + 1, (rows,), generator=g).tolist()   # noqa: E731
    t.step(draw(0, 2 * per), most)
    t.step([1] * rows, most)
    fin = (torch.rand((rows,), generator=g) < 0.4).tolist()
    t.step(draw(-2, 3 * per), most, fin)
    for _ in range(3):
        t.step(draw(0, 2), most, (torch.rand((rows,), generator=g) < 0.1).tolist())
    t.step([0] * rows, most, [True] * rows)
    assert t.count == pages and t.lengths == [0] * rows


def test_tables_refuse_in_order():
    t = TablesPair(5, 3, 6, 16)                       # 48 tokens a row, 6 pages
    got = t.step([20, 49, 40, 10, 7], 100)            # row 1 is too long for its table and asks for nothing
    assert got.granted.tolist() == [True, False, True, True, False]
    t.step([12, 1, 8, 6, 0], 100)                     # rows 0, 2, 3 need no page; none is left for row 1
    assert t.lengths == [32, 0, 48, 16, 0]
    t.step([0, 5, 0, 0, 5], 100, [False, False, True, False, False])
    t.step([1, 1, 1, 1, 1], 3)                        # places of the slot list end
    t.step([0] * 5, 0)
    t.step([3, 0, 0, 0, 0], 0)


def test_tables_in_a_replayed_graph():
    """A captured step follows the lengths by itself: the slots of every replay are the plain form's."""
    t = TablesPair(7, 5, 40, 16)
    t.step([3, 0, 15, 16, 1, 30, 2], 80)
    new, fin = i32([1, 1, 1, 1, 0, 1, 2]), torch.zeros(7, dtype=torch.bool, device=DEV)
    table0, state0 = t.gpu.block_table.clone(), (t.gpu.lengths.clone(), t.gpu.free_blocks.clone(), t.gpu.free_count.clone())
    t.gpu.step(new, max_tokens=16, finished=fin)      # warm up, then put back
    t.gpu.block_table.copy_(table0)
    for x, y in zip((t.gpu.lengths, t.gpu.free_blocks, t.gpu.free_count), state0):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = t.gpu.step(new, max_tokens=16, finished=fin)
    for turn in range(20):
        fin.copy_(torch.tensor([turn % 5 == 4] + [False] * 5 + [turn == 7], device=DEV))
        graph.replay()
        slots, pos, starts, granted, t.count = ref.tables_step(t.table, t.lengths, t.free, t.count, new.tolist(),
                                                               fin.tolist(), 16, 16)
        assert (got.slots.tolist(), got.positions.tolist()) == (slots, pos)
        assert (got.query_start.tolist(), got.granted.tolist()) == (starts, granted)
        assert t.gpu.block_table.tolist() == t.table


def test_tables_of_nothing():
    t = BlockTables.allocate(requests=0, blocks_per_request=0, blocks=3, device=DEV)
    got = t.step(i32([]), max_tokens=2)
    assert got.slots.tolist() == [-1, -1] and got.query_start.tolist() == [0] and t.free_count.tolist() == [3]


# ---- append and read --------------------------------------------------------------


class Cache:
    """A one-layer PagedKVCache (layer 1 of 2) beside numpy copies of its tensors."""

    def __init__(self, pages, heads, dim, block, seed=0, fill=True):
        self.gpu = PagedKVCache.allocate(layers=2, blocks=pages, kv_heads=heads, head_dim=dim, block_size=block, device=DEV)
        g = gen(seed)
        if fill:   # what earlier tokens left
            for t in (self.gpu.k_codes, self.gpu.v_codes):
                t.copy_(torch.randn(t.shape, generator=g).mul_(40).round_().clamp_(-127, 127).to(torch.int8))
            self.gpu.k_scales.copy_(torch.rand(self.gpu.k_scales.shape, generator=g) * 0.03 + 0.005)
            self.gpu.v_scales.copy_(torch.rand(self.gpu.v_scales.shape, generator=g) * 0.03 + 0.005)
        self.other = [t[0].clone() for t in self.tensors()]
        self.pull()

    def tensors(self):
        return self.gpu.k_codes, self.gpu.v_codes, self.gpu.k_scales, self.gpu.v_scales

    def pull(self):
        self.k, self.v, self.ks, self.vs = (t[1].cpu().numpy().copy() for t in self.tensors())

    def append(self, key, value, slots):
        self.gpu.append(1, key, value, i32(slots))
        torch.cuda.synchronize()

    def check(self):
        """The whole layer equals the plain form's, bit for bit, and the other layer is as it was."""
        for name, t, want in zip(("k", "v", "ks", "vs"), self.tensors(), (self.k, self.v, self.ks, self.vs)):
            got = t[1].cpu().numpy()
            assert np.array_equal(got, want), (name, np.argwhere(got != want)[:5])
        for t, o in zip(self.tensors(), self.other):
            assert torch.equal(t[0], o)


def finite(x):
    return torch.nan_to_num(x, nan=0.0).float().numpy()


def rows_of(shape, dtype, seed, spread=1.0):
    g = gen(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:2] + (1,), generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,block", [(2, 128, 64), (3, 64, 16), (1, 128, 32), (2, 64, 128)])
def test_append_equals_the_plain_form(heads, dim, block, dtype):
    """Prompts at odd offsets, then single tokens: codes and scales bit for bit, nothing else touched."""
    pages = 12
    c = Cache(pages, heads, dim, block, seed=dim + block)
    order = torch.randperm(pages, generator=gen(3)).tolist()
    at = lambda seq, pos: order[(seq * pages // 3 + pos // block) % pages] * block + pos % block   # noqa: E731
    plan = [[at(0, p) for p in range(0, 37)] + [at(1, p) for p in range(3, 3 + 13)] + [at(2, p) for p in range(16, 20)],
            [at(0, 37), at(1, 16), at(2, 20)], [at(0, 38), -1, at(2, 21), -7], [at(0, 39), at(1, 17), at(1, 18)],
            [-1], [at(0, p) for p in range(40, 40 + 2 * block)]]
    # the last token of the list may be the first of its unit, and the list of one entry
    plan.append([at(1, 32)])
    for i, slots in enumerate(plan):
        k, v = (rows_of((len(slots), heads, dim), dtype, 10 * i + j) for j in (0, 1))
        c.append(k.to(DEV), v.to(DEV), slots)
        ref.append(finite(k), c.k, c.ks, slots, False)
        ref.append(finite(v), c.v, c.vs, slots, True)
        c.check()


def test_append_strided_inputs_and_bad_slots():
    """Views of a stacked projection; slots past the cache are skipped, a slot named twice keeps the later token."""
    c = Cache(3, 2, 128, 32)
    qkv = rows_of((6, 10, 128), torch.bfloat16, 5).to(DEV)
    k, v = qkv[:, 4:6], qkv[:, 7:9]
    for slots in ([32, 33, 33, 34, 96, 2 ** 31 - 1], [-(2 ** 31), 5, 5, 5, 4, 6], [95, 0, 1, 16, 17, 48]):
        c.append(k, v, slots)
        ref.append(finite(k.cpu()), c.k, c.ks, slots, False)
        ref.append(finite(v.cpu()), c.v, c.vs, slots, True)
        c.check()


def test_append_one_slot_named_a_hundred_times():
    c = Cache(2, 1, 64, 16)
    k, v = rows_of((100, 1, 64), torch.float16, 1), rows_of((100, 1, 64), torch.float16, 2)
    slots = [18] * 70 + [19] * 30
    c.append(k.to(DEV), v.to(DEV), slots)
    kk, vv = k.clone(), v.clone()   # the others count neither in codes nor in scales
    ref.append(finite(kk), c.k, c.ks, slots, False)
    ref.append(finite(vv), c.v, c.vs, slots, True)
    c.check()


@pytest.mark.parametrize("dim,heads,tokens", [(128, 150, 15), (64, 150, 29), (128, 150, 60), (64, 150, 250), (128, 9, 3700)])
def test_append_long_lists_of_mixed_runs(dim, heads, tokens):
    """Runs of 1 to 70 slots from any offset, doubled slots, skipped entries: waves take several units, or none."""
    block, pages = 16, tokens // 4 + 80
    c = Cache(pages, heads, dim, block, seed=tokens)
    g, slots, page = gen(tokens), [], 0
    while len(slots) < tokens:
        n, at = (int(torch.randint(1, 71, (), generator=g)) if torch.rand((), generator=g) < 0.4 else 1), \
            int(torch.randint(0, 16, (), generator=g))
        run_ = [page * block + at + i for i in range(n)]
        page = run_[-1] // block + 1                 # a unit is in one run only
        kind = int(torch.randint(0, 4, (), generator=g))
        slots += run_ + ([run_[-1]] * 2 if kind == 0 else [-1] if kind == 1 else [])
    slots = [x if x < pages * block else -1 for x in slots[:tokens]]
    k, v = (rows_of((tokens, heads, dim), torch.bfloat16, tokens + i, spread=4.0) for i in range(2))
    c.append(k.to(DEV), v.to(DEV), slots)
    ref.append(finite(k), c.k, c.ks, slots, False)
    ref.append(finite(v), c.v, c.vs, slots, True)
    c.check()


def test_sizes_that_do_not_fit_and_rows_that_overlap():
    lengths, news = [40, 70], [3, 5]
    c, table, q, starts, scale = attention_case(lengths, news, 4, 2, 64, 16, torch.bfloat16, seed=5)
    want = run(c, table, lengths, q, starts, scale)
    table, lengths, starts = i32(table), i32(lengths), i32(starts)
    got = c.gpu.attend(1, q.to(DEV), table, lengths, scale=scale, query_start=starts, max_query=2 ** 32 + 1)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="overlap"):      # one row for all sequences
        c.gpu.attend(1, q.to(DEV), table[:1].expand(2, -1), lengths, scale=scale, query_start=starts, max_query=5)
    t = TablesPair(2, 2, 4, 16)
    for most in (-1, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="max_tokens"):
            t.gpu.step(i32([1, 1]), max_tokens=most)


def test_the_tensors_stay_the_objects_own():
    c, t = Cache(2, 1, 64, 16), TablesPair(2, 2, 4, 16)
    for obj, name in ((c.gpu, "k_codes"), (c.gpu, "v_scales"), (t.gpu, "lengths"), (t.gpu, "block_table")):
        with pytest.raises(AttributeError):
            setattr(obj, name, getattr(obj, name).clone())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_not_finite_zero_and_tiny(dtype):
    c = Cache(2, 2, 128, 16, fill=False)
    big = torch.finfo(dtype).max
    k = rows_of((32, 2, 128), dtype, 8)
    k[0, 0, 5], k[1, 0, 6], k[2, 0, 7] = float("nan"), float("inf"), -float("inf")
    k[16:, 1] = 0                                  # a unit of zeros: scale 0, codes 0
    k[16:, 0] = 1e-39 if dtype == torch.bfloat16 else 6e-8
    v = torch.full_like(k, big)
    v[3, 1, 2] = -big
    c.append(k.to(DEV), v.to(DEV), list(range(32)))
    ref.append(finite(k), c.k, c.ks, list(range(32)), False)
    ref.append(finite(v), c.v, c.vs, list(range(32)), True)
    c.check()
    assert c.ks[1, 1, 0] == 0 and not c.k[1, 1, 0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_read_gives_the_codes_back(dim, dtype):
    c = Cache(5, 3, dim, 32, seed=dim)
    g = gen(4)
    lists = [[7], list(range(20, 75)), torch.randint(0, 160, (83,), generator=g).tolist(),
             [0, -1, 159, 160, 2 ** 31 - 1, 3, 3], [-1] * 17]
    for slots in lists:
        k, v = c.gpu.read(1, i32(slots), dtype)
        ok = np.array([0 <= s < 160 for s in slots])
        at = np.where(ok, slots, 0)
        for got, codes, scales, tr in ((k, c.k, c.ks, False), (v, c.v, c.vs, True)):
            want = ref.values(codes, scales, at, tr) * ok[:, None, None]
            # the fp32 product is rounded once more to the 16-bit type
            want = torch.from_numpy(want.astype(np.float32)).to(dtype)
            assert torch.equal(got.cpu(), want)


# ---- attention ------------------------------------------------------------------


def attention_case(lengths, news, hq, hkv, dim, block, dtype, seed, scale=None, q_gain=1.5, pages_more=3):
    """Random codes under random pages; returns (cache, table, q, starts, scale)."""
    g = gen(seed)
    count = [-(-n // block) for n in lengths]
    pages = sum(count) + pages_more
    c = Cache(pages, hkv, dim, block, seed=seed)
    order = torch.randperm(pages, generator=g).tolist()
    width = max(count + [1]) + 1
    table = [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in count]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = (torch.randn((starts[-1], hq, dim), generator=g) * q_gain).to(dtype)
    return c, table, q, starts, dim ** -0.5 if scale is None else scale


def check_attention(c, table, lengths, q, starts, scale, got):
    dtype = q.dtype
    want, tol = ref.attend(q.double().numpy(), c.k, c.v, c.ks, c.vs, table, lengths, starts, scale, dtype)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(err).all() and (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:5])


def run(c, table, lengths, q, starts, scale, **kw):
    return c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale, query_start=i32(starts),
                        max_query=max(1, max(b - a for a, b in zip(starts, starts[1:]))), **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,block", [(6, 2, 128, 64), (8, 8, 128, 16), (16, 1, 64, 32), (5, 1, 128, 128),
                                              (14, 2, 64, 16), (40, 1, 128, 16)])
def test_single_tokens(hq, hkv, dim, block, dtype):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 255, 257, 700, 1]
    n = len(lengths)
    c, table, q, _, scale = attention_case(lengths, [1] * n, hq, hkv, dim, block, dtype, seed=hq + dim)
    got = c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale)
    check_attention(c, table, lengths, q, list(range(n + 1)), scale, got)
    assert not got[1].any()
    again = c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale, max_length=700)
    check_attention(c, table, lengths, q, list(range(n + 1)), scale, again)
    assert torch.equal(got, c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale))   # reproducible


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,news,hq,hkv,dim,block", [
    ([300, 40, 7, 0, 65], [2, 4, 1, 0, 3], 6, 2, 128, 16),        # a few guessed tokens
    ([70, 33, 128, 1], [70, 33, 128, 1], 6, 2, 128, 32),          # whole prompts
    ([700, 513], [150, 5], 3, 1, 128, 64),                        # a chunk over what came before
    ([90, 200], [90, 130], 8, 8, 64, 16), ([129, 64, 300], [43, 44, 45], 12, 4, 64, 64),
    ([50, 20], [50, 20], 40, 2, 128, 16), ([2, 5], [4, 5], 4, 2, 128, 16)])   # more queries than tokens: zeros
def test_prompts(lengths, news, hq, hkv, dim, block, dtype):
    c, table, q, starts, scale = attention_case(lengths, news, hq, hkv, dim, block, dtype, seed=sum(lengths))
    check_attention(c, table, lengths, q, starts, scale, run(c, table, lengths, q, starts, scale))


def test_a_long_sequence_split_and_joined():
    """Both kernels' splits: one token and a chunk of 40 over 9000 tokens, odd lengths on either side of a split."""
    for news in ([1, 1], [40, 1]):
        c, table, q, starts, scale = attention_case([9000, 513], news, 4, 2, 128, 64, torch.bfloat16, seed=5)
        got = run(c, table, [9000, 513], q, starts, scale)
        check_attention(c, table, [9000, 513], q, starts, scale, got)


def test_pages_outside_the_cache_are_left_out():
    lengths = [200, 70, 40]
    for news in ([1, 1, 1], [60, 70, 1]):
        c, table, q, starts, scale = attention_case(lengths, news, 4, 2, 128, 16, torch.bfloat16, seed=9)
        table[0][3], table[0][11], table[1][0], table[1][4] = -1, 2 ** 31 - 1, c.gpu.pages, -(2 ** 31)
        table[2] = [-1] * len(table[2])                       # a sequence without a single page
        check_attention(c, table, lengths, q, starts, scale, run(c, table, lengths, q, starts, scale))


def test_rows_and_lengths_outside_what_is_asked():
    """Rows behind the last sequence stay; lengths past the bound count as the bound; negative ones as none."""
    lengths = [100, 64]
    c, table, q, starts, scale = attention_case(lengths, [3, 2], 4, 2, 128, 32, torch.float16, seed=2)
    q = torch.cat([q, q[:3]])
    out = torch.full((8, 4, 128), 7.0, dtype=torch.float16, device=DEV)
    run(c, table, lengths, q, starts, scale, out=out)
    assert bool((out[5:] == 7).all())
    check_attention(c, table, lengths, q[:5], starts, scale, out[:5])
    got = run(c, table, [2 ** 31 - 1, 64], q, starts, scale, max_length=96)
    check_attention(c, table, [96, 64], q[:5], starts, scale, got[:5])
    assert not got[5:].any()
    got = c.gpu.attend(1, q[:2].to(DEV), i32(table), i32([-5, 64]), scale=scale)
    check_attention(c, table, [0, 64], q[:2], [0, 1, 2], scale, got)
    # queries past max_query of their sequence are not answered, the others keep their positions
    out.fill_(7.0)
    c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale, query_start=i32(starts), max_query=2, out=out)
    want, tol = ref.attend(q[:5].double().numpy(), c.k, c.v, c.ks, c.vs, table, lengths, starts, scale, torch.float16)
    err = np.abs(out[:5].double().cpu().numpy() - want)
    assert (err[[0, 1, 3, 4]] <= tol[[0, 1, 3, 4]]).all() and bool((out[2] == 7).all())


@pytest.mark.parametrize("lengths,news,before,behind", [([100, 64], [3, 2], 0, 3), ([100, 64], [3, 2], 2, 0), ([90, 80, 70], [60, 0, 50], 3, 200),
                                                        ([5000], [4], 1, 70), ([5000], [150], 5, 9), ([0, 3], [0, 0], 0, 6)])
def test_a_new_output_is_zero_where_no_query_is(lengths, news, before, behind):
    """Rows before the first and behind the last sequence, and past max_query, in memory that held something else."""
    c, table, q, starts, scale = attention_case(lengths, news, 6, 2, 128, 32, torch.bfloat16, seed=9)
    filler = lambda n: torch.full((n, 6, 128), 2.0, dtype=q.dtype)   # noqa: E731
    q = torch.cat([filler(before), q, filler(behind)])
    starts = [s + before for s in starts]
    longest = max(1, max(news))
    for most in {longest, max(1, longest - 1)}:
        torch.full((q.numel(),), float("nan"), dtype=q.dtype, device=DEV)    # what a new tensor may find
        got = c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale, query_start=i32(starts), max_query=most)
        kept = torch.full((len(q), 6, 128), 7.0, dtype=q.dtype, device=DEV)
        c.gpu.attend(1, q.to(DEV), i32(table), i32(lengths), scale=scale, query_start=i32(starts), max_query=most, out=kept)
        none = torch.ones(len(q), dtype=torch.bool)
        for a, n in zip(starts, news):
            none[a:a + min(n, most)] = False
        assert bool((kept[none.to(DEV)] == 7).all()) and not got[none.to(DEV)].any()
        assert torch.equal(got[~none.to(DEV)], kept[~none.to(DEV)])


def test_strided_queries_and_outputs():
    lengths = [130, 17]
    c, table, q, starts, scale = attention_case(lengths, [1, 1], 6, 2, 128, 16, torch.bfloat16, seed=12)
    qkv = torch.zeros((2, 10, 128), dtype=torch.bfloat16, device=DEV)
    qkv[:, :6] = q.to(DEV)
    out = torch.zeros((2, 9, 128), dtype=torch.bfloat16, device=DEV)
    c.gpu.attend(1, qkv[:, :6], i32(table), i32(lengths), scale=scale, out=out[:, 2:8])
    check_attention(c, table, lengths, q, starts, scale, out[:, 2:8])
    assert not out[:, :2].any() and not out[:, 8:].any()
    wide = torch.full((2, len(table[0]) + 5), -9, dtype=torch.int32, device=DEV)
    wide[:, :len(table[0])] = i32(table)
    got = c.gpu.attend(1, q.to(DEV), wide[:, :len(table[0])], i32(lengths), scale=scale)
    assert torch.equal(got, out[:, 2:8])


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 50, 33]])
def test_values_of_every_magnitude(news):
    """Loud and faint units side by side, units of zeros, a negative scale, outliers in the query."""
    lengths = [140, 50, 33]
    c, table, q, starts, _ = attention_case(lengths, news, 4, 2, 128, 16, torch.bfloat16, seed=21, q_gain=0.5)
    g = gen(3)
    vs = c.gpu.v_scales[1]
    vs.copy_(torch.exp2(torch.randint(-30, 12, vs.shape, generator=g).float()))
    zero = torch.rand(vs.shape, generator=g) < 0.3
    vs[zero.to(DEV)] = 0
    c.gpu.v_codes[1][zero.to(DEV)] = 0
    ks = c.gpu.k_scales[1]
    none = (torch.rand(ks.shape, generator=g) < 0.2).to(DEV)
    ks[none] = 0
    c.gpu.k_codes[1][none] = 0
    c.pull()
    q[:, :, 7] *= 64
    q[0, 1] *= 2.0 ** -60
    q[0, 2] = 0
    for scale in (0.05, -0.05, 0.0):
        check_attention(c, table, lengths, q, starts, scale, run(c, table, lengths, q, starts, scale))


def test_a_query_that_is_not_finite_spoils_its_own_row_only():
    lengths = [60, 60]
    for news in ([1, 1], [40, 30]):
        c, table, q, starts, scale = attention_case(lengths, news, 4, 2, 128, 16, torch.bfloat16, seed=31)
        clean = run(c, table, lengths, q, starts, scale)
        q[1, 2, 5] = float("nan")
        got = run(c, table, lengths, q, starts, scale)
        keep = torch.ones(q.shape[:2], dtype=torch.bool)
        keep[1, 2] = False
        assert torch.equal(got[keep.to(DEV)], clean[keep.to(DEV)]) and bool(got[1, 2].isnan().any())


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes, the sequence in its last pages."""
    pages, hkv, block = 9000, 64, 64                   # 4.7 GB of key codes and as much of values
    big = PagedKVCache(torch.empty((1, pages, hkv, 4, 16, 128), dtype=torch.int8, device=DEV),
                       torch.empty((1, pages, hkv, 4, 128, 16), dtype=torch.int8, device=DEV),
                       torch.zeros((1, pages, hkv, 4), device=DEV), torch.zeros((1, pages, hkv, 4), device=DEV))
    k, v = (rows_of((130, hkv, 128), torch.bfloat16, s, 0.2).to(DEV) for s in (1, 2))
    slots = [(pages - 1 - p // block) * block + p % block for p in range(130)]
    big.append(0, k, v, i32(slots))
    small = PagedKVCache.allocate(layers=1, blocks=3, kv_heads=hkv, block_size=block, device=DEV)
    small.append(0, k, v, i32(list(range(130))))
    for x, y in zip(big.read(0, i32(slots), torch.bfloat16), small.read(0, i32(list(range(130))), torch.bfloat16)):
        assert torch.equal(x, y)
    q = rows_of((1, hkv, 128), torch.bfloat16, 3, 0.1).to(DEV)
    got = big.attend(0, q, i32([[pages - 1, pages - 2, pages - 3]]), i32([130]), scale=0.09)
    assert torch.equal(got, small.attend(0, q, i32([[0, 1, 2]]), i32([130]), scale=0.09))


def test_refusals_on_the_device():
    c = Cache(4, 2, 128, 16)
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV)
    table, lengths = i32([[0, 1], [2, 3]]), i32([20, 20])
    ok = dict(scale=0.1)
    for bad in (lambda: c.gpu.attend(1, q.float(), table, lengths, **ok), lambda: c.gpu.attend(1, q[:, :3], table, lengths, **ok),
                lambda: c.gpu.attend(1, q, table.long(), lengths, **ok), lambda: c.gpu.attend(1, q, table, lengths[:1], **ok),
                lambda: c.gpu.attend(1, q[:1], table, lengths, **ok), lambda: c.gpu.attend(1, q[:, :, :64], table, lengths, **ok),
                lambda: c.gpu.attend(1, q, table, lengths, scale=float("nan")),
                lambda: c.gpu.attend(1, q, table, lengths, query_start=i32([0, 1]), **ok),
                lambda: c.gpu.attend(1, q, table, lengths, out=q.half(), **ok),
                lambda: c.gpu.append(1, q, q, i32([0, 1])), lambda: c.gpu.append(1, q[:, :2], q[:, :2].half(), i32([0, 1])),
                lambda: c.gpu.append(1, q[:, :2], q[:, :2], i32([0])), lambda: c.gpu.read(1, i32([0]).long(), q.dtype),
                lambda: c.gpu.read(1, i32([0]), torch.float32),
                lambda: BlockTables.allocate(requests=1, blocks_per_request=1, blocks=1, device=DEV).step(
                    i32([1, 2]), max_tokens=1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        c.gpu.attend(2, q, table, lengths, **ok)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        c.gpu.append(1, q[:, :2].cpu(), q[:, :2], i32([0, 1]))


# ---- together -------------------------------------------------------------------


def test_serving_steps_together():
    """Admissions, decoding, a request that ends and one that takes its row: tables, append and attention as a serving
    loop runs them, every step against the plain forms on what the cache holds."""
    hq, hkv, dim, block = 6, 2, 128, 16
    t = TablesPair(3, 12, 30, block)
    c = Cache(30, hkv, dim, block, fill=False)
    steps = [([37, 20, 0], None), ([1, 1, 5], None), ([1, 1, 1], None), ([3, 50, 1], [False, True, False]),
             ([1, 0, 1], None), ([0, 1, 9], [True, False, True])]
    for i, (new, fin) in enumerate(steps):
        got = t.step(new, 96, fin)
        k, v, q = (rows_of((96, h, dim), torch.bfloat16, 100 * i + j, 0.3) for j, h in enumerate((hkv, hkv, hq)))
        c.gpu.append(1, k.to(DEV), v.to(DEV), got.slots)
        out = c.gpu.attend(1, q.to(DEV), t.gpu.block_table, t.gpu.lengths, scale=dim ** -0.5,
                           query_start=got.query_start, max_query=max(new))
        slots, starts = got.slots.tolist(), got.query_start.tolist()
        ref.append(finite(k), c.k, c.ks, slots, False)
        ref.append(finite(v), c.v, c.vs, slots, True)
        c.check()
        check_attention(c, t.table, t.lengths, q[:starts[-1]], starts, dim ** -0.5, out[:starts[-1]])
        assert not out[starts[-1]:].any()


def test_a_captured_decoding_step():
    """Tables, append and attention in one graph: every replay equals the eager step on a copy."""
    hq, hkv, dim, block, rows = 6, 2, 128, 16, 3
    def fresh():
        tables = BlockTables.allocate(requests=rows, blocks_per_request=8, blocks=20, block_size=block, device=DEV)
        cache = PagedKVCache.allocate(layers=1, blocks=20, kv_heads=hkv, head_dim=dim, block_size=block, device=DEV)
        first = tables.step(i32([14, 30, 1]), max_tokens=45)
        k = rows_of((45, hkv, dim), torch.bfloat16, 1).to(DEV)
        cache.append(0, k, k.flip(0), first.slots)
        return tables, cache
    one = i32([1] * rows)
    k, v, q = (torch.zeros((rows, h, dim), dtype=torch.bfloat16, device=DEV) for h in (hkv, hkv, hq))
    def step(tables, cache):
        got = tables.step(one, max_tokens=rows)
        cache.append(0, k, v, got.slots)
        return cache.attend(0, q, tables.block_table, tables.lengths, scale=0.1)
    step(*fresh())
    a, b = fresh(), fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*a)
    for i in range(24):
        for t, s in ((k, 1), (v, 2), (q, 3)):
            t.copy_(rows_of(tuple(t.shape), torch.bfloat16, 10 * i + s))
        graph.replay()
        want = step(*b)
        assert torch.equal(out, want), i
        assert torch.equal(a[1].k_codes, b[1].k_codes) and torch.equal(a[1].v_scales, b[1].v_scales)


def test_two_streams_at_once():
    """Calls on two streams share nothing: each has a workspace of its own."""
    lengths = [5000, 4000]
    c, table, q, starts, scale = attention_case(lengths, [1, 1], 8, 2, 128, 64, torch.bfloat16, seed=6)
    tab, lens, qd = i32(table), i32(lengths), q.to(DEV)
    other = qd.flip(0).contiguous()
    want = [c.gpu.attend(1, x, tab, lens, scale=scale) for x in (qd, other)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, (qd, other)):
            with torch.cuda.stream(s):
                got.append(c.gpu.attend(1, x, tab, lens, scale=scale))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert paged_attention_workspace(2, 2, 8, 2, 128, 1, tab.shape[1] * 64, DEV).numel() > 0
