"""The paged cache's refusals and host-side sizing: no GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tilequant_amd import _native as nat
from tilequant_amd.paged_cache import BlockTables, PagedKVCache

FAKE = 1 << 20   # a non-null, 16-byte aligned host value: every check here comes before any launch


def cache(**over):
    f = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, pages=8, kv_heads=2, head_dim=128, block=64)
    f.update(over)
    return ctypes.byref(nat.Kv8Cache(**f))


BAD_CACHES = [dict(head_dim=96), dict(block=48), dict(block=8), dict(block=2048), dict(kv_heads=0), dict(pages=-1),
              dict(pages=1 << 26), dict(k_codes=None), dict(v_scales=None)]


@pytest.mark.parametrize("over", BAD_CACHES)
def test_append_and_read_refuse_caches_they_cannot_take(over):
    lib = nat.load()
    assert lib.tq_kv8_append(cache(**over), FAKE, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -1
    assert lib.tq_kv8_read(cache(**over), FAKE, 4, 0, FAKE, 256, 128, FAKE, 256, 128, None) == -1


def test_append_and_read_refusals():
    lib = nat.load()
    assert lib.tq_kv8_append(cache(), FAKE, 256, 128, FAKE, 256, 128, 2, FAKE, 4, None) == -2     # fp32 is not taken
    assert lib.tq_kv8_append(cache(), FAKE, 256, 128, FAKE, 256, 128, 0, FAKE, -1, None) == -1
    assert lib.tq_kv8_append(cache(), None, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -1
    assert lib.tq_kv8_append(cache(), FAKE, 256, 128, FAKE, 256, 128, 0, None, 4, None) == -1
    assert lib.tq_kv8_append(cache(), FAKE + 2, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -3
    assert lib.tq_kv8_append(cache(), FAKE, 260, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -3
    assert lib.tq_kv8_append(cache(k_codes=FAKE + 8), FAKE, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -3
    assert lib.tq_kv8_append(None, FAKE, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == -1
    assert lib.tq_kv8_append(cache(), None, 256, 128, None, 256, 128, 0, None, 0, None) == 0      # nothing to do
    assert lib.tq_kv8_append(cache(pages=0), FAKE, 256, 128, FAKE, 256, 128, 0, FAKE, 4, None) == 0
    assert lib.tq_kv8_read(cache(), FAKE, 4, 2, FAKE, 256, 128, FAKE, 256, 128, None) == -2
    assert lib.tq_kv8_read(cache(), FAKE, 4, 0, FAKE, 256, 128, FAKE, 250, 128, None) == -3
    assert lib.tq_kv8_read(cache(), FAKE, 0, 0, None, 256, 128, None, 256, 128, None) == 0


def attention(cache_, *, q=FAKE, dtype=0, table=FAKE, ld=4, width=4, lengths=FAKE, starts=None, tokens=3, batch=3, heads=8,
              max_query=1, max_len=256, scale=0.1, out=FAKE, ws=None, ws_elems=0, st=1024, sh=128):
    return nat.load().tq_kv8_attention(cache_, q, st, sh, dtype, table, ld, width, lengths, starts, tokens, batch, heads,
                                       max_query, max_len, scale, out, 1024, 128, 0, ws, ws_elems, None)


def test_attention_refusals():
    for over in BAD_CACHES[:-3]:
        assert attention(cache(**over)) == -1, over
    assert attention(cache(pages=0)) == -1
    assert attention(cache(), dtype=2) == -2
    assert attention(cache(), heads=7) == -1
    assert attention(cache(kv_heads=1), heads=129) == -1
    assert attention(cache(), tokens=4) == -1                    # one query per sequence without query_start
    assert attention(cache(), max_query=2) == -1
    assert attention(cache(), ld=3) == -1
    assert attention(cache(), q=None) == -1 and attention(cache(), lengths=None) == -1
    assert attention(cache(), scale=float("nan")) == -1 and attention(cache(), scale=float("inf")) == -1
    assert attention(cache(), q=FAKE + 8) == -3 and attention(cache(), sh=124) == -3
    assert attention(cache(), tokens=0, batch=0) == 0
    # a batch of one over a long table is split, and then needs its workspace
    need = nat.load().tq_kv8_attention_workspace_elems(1, 1, 8, 2, 128, 1, 1 << 16)
    assert need > 0 and need % 130 == 0
    assert attention(cache(), tokens=1, batch=1, ld=1024, width=1024, max_len=1 << 16) == -4
    assert attention(cache(), tokens=1, batch=1, ld=1024, width=1024, max_len=1 << 16, ws=FAKE, ws_elems=need - 1) == -4


def test_tables_refusals():
    step = nat.load().tq_block_tables_step
    ok = dict(new=FAKE, fin=None, table=FAKE, ld=4, lengths=FAKE, free=FAKE, cap=8, count=FAKE, slots=FAKE, pos=FAKE,
              starts=FAKE, granted=FAKE, rows=2, width=4, block=64, most=16)
    call = lambda **o: step(*[{**ok, **o}[k] for k in ok], None)   # noqa: E731
    for bad in (dict(new=None), dict(table=None), dict(ld=3), dict(lengths=None), dict(count=None), dict(free=None),
                dict(slots=None), dict(starts=None), dict(granted=None), dict(rows=-1), dict(block=0), dict(most=-1),
                dict(width=1 << 26, ld=1 << 26), dict(cap=1 << 26)):
        assert call(**bad) == -1, bad


def test_workspace_is_none_for_what_is_not_split():
    elems = nat.load().tq_kv8_attention_workspace_elems
    assert elems(64, 64, 32, 32, 128, 1, 4096) == 0      # 2048 workgroups as it is
    assert elems(0, 1, 8, 2, 128, 1, 4096) == 0 and elems(1, 1, 7, 2, 128, 1, 4096) == 0
    assert elems(1, 1, 8, 2, 128, 1, 0) == 0


def test_no_cpu_tensors():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        BlockTables.allocate(requests=2, blocks_per_request=4, blocks=8, device="cpu")
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        PagedKVCache.allocate(layers=1, blocks=2, kv_heads=1, device="cpu")
    with pytest.raises(ValueError, match="power of two"):
        PagedKVCache.allocate(layers=1, blocks=2, kv_heads=1, block_size=48, device="cpu")
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        PagedKVCache(z((1, 2, 1, 1, 16, 64)), z(1), z(1), z(1))
