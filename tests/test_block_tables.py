"""Block tables, page table and slot map from request lengths (paging.grow_block_tables) against the
request-by-request oracle, its refusals, and a run of it with the 4-bit cache: tables, write, append,
decode, step after step."""
import ctypes

import numpy as np
import pytest
import torch

import attention
import dk_lib
import layout
import paging
from dk_lib import DecodeArgumentError
from helpers import to_np
from oracle import kv4

DEV = "cuda"


def test_oracle_by_hand():
    table = np.full((3, 4), -1)
    table[2, 0] = 9
    got = kv4.grow(table, [2, 0], [15, 0], [3, 0], [5, 6], 5, 4)
    assert got[0].tolist() == [[-1] * 4, [-1] * 4, [9, 5, -1, -1]]
    assert got[1:] == ([0, 2, 2], [9, 5, None, None], [2, 0], [0, 3, 3], [9 * 16 + 15, 80, 81, -1, -1],
                       [15, 16, 17, 0, 0])


def _args(**kw):
    a = dict(block_table=torch.zeros(4, 8, dtype=torch.int32), rows=torch.zeros(2, dtype=torch.int32),
             cached_lens=torch.zeros(2, dtype=torch.int64), new_lens=torch.ones(2, dtype=torch.int32),
             new_pages=torch.zeros(2, dtype=torch.int32), num_tokens=2, capacity=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(block_table=torch.zeros(4, 8)), dict(block_table=torch.zeros(32, dtype=torch.int32)),
    dict(block_table=torch.zeros(8, 4, dtype=torch.int32).t()),
    dict(block_table=torch.zeros(8, dtype=torch.int32).expand(4, 8)),
    dict(rows=torch.zeros(2)), dict(rows=torch.zeros(2, 1, dtype=torch.int32)),
    dict(cached_lens=torch.zeros(3, dtype=torch.int32)), dict(new_lens=torch.zeros(1, dtype=torch.int32)),
    dict(new_pages=torch.zeros(2, dtype=torch.int64)), dict(num_tokens=-1), dict(capacity=2 ** 31),
    dict(num_tokens=True), dict(capacity=2.0), dict()])        # the last: all well but for the device
def test_refusals(kw):
    with pytest.raises(DecodeArgumentError):
        paging.grow_block_tables(**_args(**kw))


def test_refuses_what_is_no_tensor():
    for name in ("block_table", "rows", "cached_lens", "new_pages"):
        with pytest.raises(TypeError):
            paging.grow_block_tables(**_args(**{name: [1, 2]}))


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), dk_lib.DK_EINVAL), (dict(blocks=1 << 27), dk_lib.DK_EINVAL),
    (dict(stride=4), dk_lib.DK_EINVAL), (dict(stride=1 << 41), dk_lib.DK_EUNSUPPORTED),
    (dict(tokens=1 << 31), dk_lib.DK_EINVAL), (dict(rows=None), dk_lib.DK_ENULL),
    (dict(table=None), dk_lib.DK_ENULL), (dict(slots=None), dk_lib.DK_ENULL),
    (dict(batch=0, rows=None), dk_lib.DK_OK)])
def test_abi_refusals(kw, code):
    a = dict(table=0x1000, stride=8, rows=0x2000, batch=2, blocks=8, slots=0x3000, tokens=2)
    a.update(kw)
    assert dk_lib.load().dk_grow_block_tables(
        a["table"], a["stride"], 4, a["blocks"], a["rows"], 0, 0x4000, 0, 0x5000, 0, 0x6000, 2, a["batch"],
        0x7000, 0x8000, 2, 0x9000, 0xa000, a["slots"], 0xb000, a["tokens"], None) == code


def _grow(table, rows, cached, added, pages, num_tokens, capacity, wide=False, **kw):
    t = lambda x, dt=torch.int32: torch.tensor(np.asarray(x), dtype=dt, device=DEV)  # noqa: E731
    dt = torch.int64 if wide else torch.int32
    dev_table = table if isinstance(table, torch.Tensor) else t(table)
    got = paging.grow_block_tables(dev_table, t(rows, dt), t(cached, dt), t(added, dt), t(pages),
                                   num_tokens, capacity, **kw)
    torch.cuda.synchronize()
    return dev_table, got


def _same(dev_table, got, want):
    table, indptr, ids, last, q_indptr, slots, pos = want
    np.testing.assert_array_equal(to_np(dev_table), table)
    for g, w in zip((got.kv_indptr, got.kv_last_page_len, got.q_indptr, got.slots, got.positions),
                    (indptr, last, q_indptr, slots, pos)):
        np.testing.assert_array_equal(to_np(g), w)
    assert got.kv_indices.shape[0] == len(ids)
    for g, w in zip(to_np(got.kv_indices), ids):
        assert w is None or g == w


@pytest.mark.gpu
@pytest.mark.parametrize("batch,cached,added,blocks,spare,wide", [
    (1, (0, 1), (1, 2), 1, 0, False), (1, (0, 1), (130000, 130001), 9000, 3, True),
    (3, (0, 40), (0, 3), 8, 0, True), (64, (1, 8000), (1, 2), 513, 5, False),
    (9, (0, 500), (33, 777), 90, -4, True), (700, (0, 300), (0, 65), 24, 1, False),
    (5, (15, 18), (0, 1), 3, 0, False)])
def test_matches_the_oracle(batch, cached, added, blocks, spare, wide):
    print(f"[case] tables {batch} {cached} {added}", flush=True)
    r = np.random.default_rng(batch)
    c = r.integers(*cached, batch)
    n = r.integers(*added, batch)
    rows = r.permutation(batch + 4)[:batch]
    need = int((-(-(c + n) // 16) - -(-c // 16)).sum())
    ids = r.permutation(batch * blocks + need + 8).astype(np.int32)
    table = np.full((batch + 4, blocks), -7, np.int32)
    for i, x in enumerate(rows):
        table[x, :-(-c[i] // 16)] = ids[i * blocks:i * blocks + -(-c[i] // 16)]
    pages = ids[batch * blocks:][:max(0, need + spare)]           # spare < 0: too few pages
    tokens, cap = int(n.sum()) + 5, int((-(-(c + n) // 16)).sum()) + 2
    want = kv4.grow(table, rows, c, n, pages, tokens, cap)
    dev, got = _grow(table, rows, c, n, pages, tokens, cap, wide)
    _same(dev, got, want)
    dev, again = _grow(dev, rows, c, n, pages, tokens, cap, wide)   # the same call again: the same
    _same(dev, again, want)


@pytest.mark.gpu
def test_bad_requests_have_no_pages_and_short_outputs_are_not_overrun():
    table = np.arange(4 * 3, dtype=np.int32).reshape(4, 3)
    rows = [-1, 1, 9, 2, 3, 0, 2 ** 31 - 1]
    cached, added = [4, 40, 4, -3, 10, 20, 0], [2, 9, 1, 2, -5, 4, 3]     # 40 + 9 > 48
    want = kv4.grow(table, rows, cached, added, [50, 51], 22, 4)
    dev, got = _grow(table, rows, cached, added, [50, 51], 22, 4)
    _same(dev, got, want)
    # lengths near int64's end, in int64
    big = 2 ** 63 - 1
    want = kv4.grow(table, [1, 2], [big, 1], [1, 1], [], 3, 2)
    _same(*_grow(table, [1, 2], [big, 1], [1, 1], [], 3, 2, wide=True), want)
    # fewer entries than the tables have: the rest is dropped, nothing lies behind them
    out = paging.StepTables(*(torch.full((n,), -99, dtype=torch.int32, device=DEV)
                              for n in (3, 8, 2, 3, 8, 8)))
    dev, got = _grow(table, [1, 2], [30, 17], [4, 2], [70, 71], 3, 2, out=out)
    want = kv4.grow(table, [1, 2], [30, 17], [4, 2], [70, 71], 6, 5)
    assert to_np(got.kv_indptr).tolist() == want[1] and to_np(got.q_indptr).tolist() == want[4]
    assert to_np(out.kv_indices).tolist() == want[2][:2] + [-99] * 6
    assert to_np(out.slots).tolist() == want[5][:3] + [-99] * 5
    # an empty batch
    t = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    got = paging.grow_block_tables(t, e, e, e, e, 3, 0)
    assert to_np(got.kv_indptr).tolist() == [0] and to_np(got.slots).tolist() == [-1] * 3


@pytest.mark.gpu
def test_a_view_of_a_wider_table_and_a_captured_step():
    wide = torch.full((6, 12), -1, dtype=torch.int32, device=DEV)
    view = wide[:, 2:9]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    rows, cached, added, pages = t([4, 1]), t([0, 0]), t([20, 3]), t([30, 31, 32, 33])
    out = paging.StepTables(*(torch.zeros(n, dtype=torch.int32, device=DEV) for n in (3, 20, 2, 3, 40, 40)))
    graph = torch.cuda.CUDAGraph()
    paging.grow_block_tables(view, rows, cached, added, pages, 40, 20, out=out)
    wide.fill_(-1)
    with torch.cuda.graph(graph):
        paging.grow_block_tables(view, rows, cached, added, pages, 40, 20, out=out)
    have = np.full((6, 7), -1)
    c = np.array([0, 0])
    free = 30
    for n in ([20, 3], [1, 1], [0, 40], [12, 5]):
        n = np.array(n)
        need = int((-(-(c + n) // 16) - -(-c // 16)).sum())
        hand = list(range(free, free + need)) + [-1] * (4 - need)
        cached.copy_(t(c.tolist()))
        added.copy_(t(n.tolist()))
        pages.copy_(t(hand))
        graph.replay()
        torch.cuda.synchronize()
        want = kv4.grow(have, [4, 1], c, n, hand, 40, 20)
        _same(view, out, want)
        have, c, free = want[0], c + n, free + need
    assert (to_np(wide)[:, :2] == -1).all() and (to_np(wide)[:, 9:] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,hq,hkv", [(torch.float16, 128, 8, 2), (torch.bfloat16, 64, 16, 2)])
def test_a_serving_run_prefill_then_decode_steps(dtype, d, hq, hkv):
    """Requests of unequal prompts: tables, the cache write and decode over it, then steps of one
    token each, checked against the same history kept in float64."""
    print(f"[case] serving {dtype} {d}", flush=True)
    r = np.random.default_rng(d)
    prompts = [5, 31, 70]
    b, pool = len(prompts), 40
    cache = layout.alloc_kv4_cache(pool, hkv, d, device=DEV)
    table = torch.full((5, 16), -1, dtype=torch.int32, device=DEV)
    free = list(r.permutation(pool))
    rows = torch.tensor([3, 0, 4], device=DEV)
    inv = paging.rope_inv_freq(d)
    cached = np.zeros(b, int)
    eps = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    for step in range(5):
        new = np.array(prompts) if step == 0 else np.ones(b, int)
        need = int((-(-(cached + new) // 16) - -(-cached // 16)).sum())
        pages = torch.tensor([free.pop() for _ in range(need)], dtype=torch.int32, device=DEV)
        n = int(new.sum())
        st = paging.grow_block_tables(table, rows, torch.from_numpy(cached).to(DEV),
                                      torch.from_numpy(new).to(DEV), pages, n + 2,
                                      int((-(-(cached + new) // 16)).sum()))
        q, k, v = (torch.from_numpy(r.standard_normal((n + 2, h, d))).to(dtype).to(DEV)
                   for h in (hq, hkv, hkv))
        paging.write_kv4(k, v, cache, st.slots, q=q, inv_freq=inv, positions=st.positions)
        ends = st.q_indptr[1:].long() - 1
        out = attention.decode_attention(q[ends].contiguous(), cache, st.kv_indptr, st.kv_indices,
                                         st.kv_last_page_len, split_kv=0)
        torch.cuda.synchronize()
        cached = cached + new
        want, size, big = kv4.decode(to_np(q[ends].double()), to_np(cache), to_np(st.kv_indptr),
                                     to_np(st.kv_indices), to_np(st.kv_last_page_len))
        assert to_np(st.kv_last_page_len).tolist() == [(c - 1) % 16 + 1 for c in cached]
        weight = 2 * (size * 2.0 ** -14 + 2.0 ** -15)
        assert (np.abs(to_np(out.double()) - want) <=
                eps * np.abs(want) * (1 + weight) + weight * (big + np.abs(want)) + 2.0 ** -25).all()
        # the new tokens' rows are what the write holds for them
        uk, uv = kv4.unpack(to_np(cache), d)
        at = to_np(st.slots)[:n]
        np.testing.assert_array_equal(uv[at // 16, :, at % 16], kv4.held(to_np(v[:n].double())))
