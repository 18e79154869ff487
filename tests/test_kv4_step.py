"""A step over the 4-bit cache as a serving loop runs it: captured into a HIP graph and replayed beside
eager work, on other streams, two at once, and through the automatic schedules of every kind of batch."""
import numpy as np
import pytest
import torch

import attention
import extend
import layout
import paging
from helpers import to_np
from oracle import kv4
from test_kv4 import EPS, _decode_case

DEV = "cuda"
pytestmark = pytest.mark.gpu


class Loop:
    """Three requests' caches, tables and lengths; step() adds one token to each and attends to all."""

    def __init__(self, hq=8, hkv=2, d=64, dtype=torch.bfloat16, seed=0):
        self.r = np.random.default_rng(seed)
        self.hq, self.hkv, self.d, self.dtype = hq, hkv, d, dtype
        self.cache = layout.alloc_kv4_cache(40, hkv, d, device=DEV)
        self.table = torch.full((5, 12), -1, dtype=torch.int32, device=DEV)
        self.rows = torch.tensor([3, 0, 4], device=DEV)
        self.cached = torch.tensor([0, 0, 0], device=DEV)
        self.one = torch.ones(3, dtype=torch.int64, device=DEV)
        self.ids = torch.randperm(40, device=DEV).to(torch.int32)
        self.pages = torch.empty(3, dtype=torch.int32, device=DEV)   # the ids a step hands out, in order
        self.inv = paging.rope_inv_freq(d)
        self.t = paging.StepTables(*(torch.zeros(n, dtype=torch.int32, device=DEV)
                                     for n in (4, 36, 3, 4, 3, 3)))
        self.q, self.k, self.v = (self.rand(3, h) for h in (hq, hkv, hkv))
        self.used = 0

    def rand(self, n, h):
        return torch.from_numpy(self.r.standard_normal((n, h, self.d))).to(self.dtype).to(DEV)

    def prefill(self, lens):
        n, need = sum(lens), sum(-(-x // 16) for x in lens)
        new = torch.tensor(lens, device=DEV)
        t = paging.grow_block_tables(self.table, self.rows, self.cached, new, self.ids[:need], n, need)
        self.used = need
        q, k, v = (self.rand(n, h) for h in (self.hq, self.hkv, self.hkv))
        paging.write_kv4(k, v, self.cache, t.slots, q=q, inv_freq=self.inv, positions=t.positions)
        out = extend.extend_attention_kv4(q, self.cache, self.table, [3, 0, 4], lens, lens)
        self.cached += new
        return out

    def feed(self):
        """The next step's inputs, into the buffers that a graph reads."""
        for x in (self.q, self.k, self.v):
            x.copy_(self.rand(3, x.shape[1]))
        need = int((self.cached % 16 == 0).sum())
        self.pages[:need] = self.ids[self.used:self.used + need]
        self.used += need

    def step(self):
        t = paging.grow_block_tables(self.table, self.rows, self.cached, self.one, self.pages, 3, 36,
                                     out=self.t)
        q = self.q.clone()
        paging.write_kv4(self.k, self.v, self.cache, t.slots, q=q, inv_freq=self.inv, positions=t.positions)
        out = attention.decode_attention(q, self.cache, t.kv_indptr, t.kv_indices, t.kv_last_page_len,
                                         split_kv=0, max_pages_per_seq=12)
        k, v = paging.read_kv4(self.cache, t.slots, self.dtype)
        self.cached += 1
        return out, k, v


@pytest.mark.parametrize("d,hq,hkv,dtype", [(64, 8, 2, torch.bfloat16), (128, 4, 4, torch.float16)])
def test_a_captured_step_replays_as_the_eager_one(d, hq, hkv, dtype):
    a, b = (Loop(hq, hkv, d, dtype, seed=5) for _ in range(2))
    b.ids.copy_(a.ids)
    for x in (a, b):
        x.prefill([17, 40, 31])
    # capture steps nothing: the buffers' state is put back afterwards
    state = [x.clone() for x in (a.cache, a.table, a.cached)]
    a.feed()
    a.used -= int((a.cached % 16 == 0).sum())
    a.r = np.random.default_rng(99)
    b.r = np.random.default_rng(99)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = a.step()
    for x, y in zip((a.cache, a.table, a.cached), state):
        x.copy_(y)
    for step in range(20):                                   # past a page's end in every request
        a.feed()
        b.feed()
        g.replay()
        want = b.step()
        torch.cuda.synchronize()
        for x, y in zip((*outs, a.cache, a.table, a.cached), (*want, b.cache, b.table, b.cached)):
            assert torch.equal(x, y), step


@pytest.mark.parametrize("d", [64, 128])
def test_captured_prefill_split_and_dealt(d):
    """Captured prefill calls whose keys are split (a workspace of the graph's own) and whose tiles are
    dealt out, replayed with other inputs."""
    loop = Loop(8, 2, d, torch.float16, seed=d)
    loop.table = torch.arange(60, dtype=torch.int32, device=DEV).view(1, 60).repeat(2, 1)
    loop.cache = layout.alloc_kv4_cache(60, 2, d, device=DEV)
    k = loop.rand(960, 2)
    paging.write_kv4(k, loop.rand(960, 2), loop.cache, torch.arange(960, device=DEV))
    graphs = []
    for rows, new, alls in (([0], [5], [955]), ([0, 1], [300, 210], [300, 700])):
        q = loop.rand(sum(new), 8)
        call = lambda q=q, a=(rows, new, alls): extend.extend_attention_kv4(  # noqa: E731
            q, loop.cache, loop.table, *a)
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, q, out, call))
    for step in range(3):
        for g, q, out, call in graphs:
            q.copy_(loop.rand(*q.shape[:2]))
            g.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(out, want), step


def test_two_streams_at_once():
    """Calls on two streams, their scratch and outputs apart: the same as one after the other."""
    loops = [Loop(8, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    keys = [layout.alloc_kv4_cache(130, 2, 128, device=DEV) for _ in loops]
    table = torch.arange(130, dtype=torch.int32, device=DEV).view(1, 130)
    jobs = []
    for loop, cache in zip(loops, keys):
        paging.write_kv4(loop.rand(2080, 2), loop.rand(2080, 2), cache, torch.arange(2080, device=DEV))
        q = loop.rand(6, 8)
        jobs.append(lambda q=q, c=cache: (
            extend.extend_attention_kv4(q, c, table, [0], [6], [2078]),
            attention.decode_attention(q[:1], c, torch.tensor([0, 130], dtype=torch.int32, device=DEV), table[0],
                                       torch.tensor([7], dtype=torch.int32, device=DEV), split_kv=0),
            *paging.read_kv4(c, torch.arange(50, 90, device=DEV))))
    want = [[x.clone() for x in job()] for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, job in zip(streams, jobs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(job())
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


# Batches that the automatic schedule treats differently: short (one pass), near-uniform ones of few and of
# many sequences (parts), ragged ones (ranges); lengths in tokens
BATCHES = [
    ([500] * 3, 8, 2, 128), ([1] * 40, 8, 8, 64), ([1100] * 2, 8, 2, 128), ([2000] * 20, 32, 8, 64),
    ([1500, 1600] * 8, 16, 8, 256), ([5000], 64, 8, 128), ([3000, 20, 1, 0, 900, 40, 2000], 32, 8, 128),
    ([1050] * 130, 4, 2, 64), ([4000, 3800, 3900], 20, 4, 128),
]


def _random_case(lens, hq, hkv, d):
    """Random codes under scales of 2^-6 .. 2^-2, without quantising values (which takes long)."""
    r = np.random.default_rng(len(lens) + d)
    blocks = [-(-n // 16) for n in lens]
    pool = sum(blocks) + 3
    raw = r.integers(0, 256, (pool, hkv, 17 * d), dtype=np.uint8)
    raw[:, :, 16 * d:] = r.integers(121, 126, (pool, hkv, d), dtype=np.uint8)
    ids = r.permutation(pool)[:sum(blocks)].astype(np.int32)
    ip = np.r_[0, np.cumsum(blocks)].astype(np.int32)
    last = np.array([n - 16 * (p - 1) if p else 0 for n, p in zip(lens, blocks)], np.int32)
    q = torch.from_numpy(r.standard_normal((len(lens), hq, d))).to(torch.bfloat16).to(DEV)
    return q, torch.from_numpy(raw).to(DEV), raw, ip, ids, last


@pytest.mark.parametrize("lens,hq,hkv,d", BATCHES)
def test_the_automatic_schedules(lens, hq, hkv, d):
    q, cache, raw, ip, ids, last = _random_case(lens, hq, hkv, d)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    spare = torch.cat([tabs[1], torch.full((3 * len(ids) + 5,), 2 ** 30, dtype=torch.int32, device=DEV)])
    hint = attention.plan_hint(ip)
    few = min(len(lens), 4)                                  # checked against the oracle, the others among them
    held = {w: kv4.decode(to_np(q[:few].double()), raw, ip[:few + 1], ids[:ip[few]], last[:few], window=w)
            for w in (0, 1300)}
    first = {}
    for kw in (dict(max_pages_per_seq=hint), dict(), dict(max_pages_per_seq=1),
               dict(max_pages_per_seq=4 * hint), dict(max_pages_per_seq=hint, window=1300),
               dict(max_pages_per_seq=hint, waves_per_cu=4)):
        for table in (tabs[1], spare):
            out = attention.decode_attention(q, cache, tabs[0], table, tabs[2], split_kv=0, **kw)
            got, window = to_np(out.double()), kw.get("window", 0)
            want, size, big = held[window]
            weight = 2 * (size * 2.0 ** -14 + 2.0 ** -15)    # as in test_kv4._check
            tol = EPS[torch.bfloat16] * np.abs(want) * (1 + weight) + weight * (big + np.abs(want)) + 2.0 ** -25
            assert (np.abs(got[:few] - want) <= tol).all(), kw
            # two schedules' results are each within the tolerance of the same value
            other = first.setdefault(window, got)
            tol = 2 * EPS[torch.bfloat16] * np.abs(other) + 4 * weight * (big + np.abs(other)) + 2.0 ** -24
            assert np.isfinite(got).all() and (np.abs(got - other) <= 1.1 * tol).all(), kw


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (16, 2, 128), (16, 1, 256), (4, 2, 128), (20, 4, 64)])
def test_nan_values_in_decode(hq, hkv, d):
    """A value block with the NaN scale: NaN in its dims for the heads that read it; every other output
    keeps its bits. One behind the last token, or before the window, reaches nothing."""
    lens, g = [90, 300, 33], hq // hkv
    q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, torch.float16, seed=d)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    sp = kv4._places(d)[2]
    bad = raw.copy()
    hit = np.zeros((3, hq, d), bool)
    for b, tok, kvh, block in ((0, 3, 0, 0), (0, 89, hkv - 1, 1), (1, 150, 0, d // 32 - 1), (2, 33, 0, 0), (2, 47, 0, 1)):
        bad[ids[ip[b] + tok // 16], kvh, sp[tok % 16, block] + d // 2] = 255
        if tok < lens[b]:
            hit[b, g * kvh:g * (kvh + 1), 32 * block:32 * block + 32] = True
    hit = torch.from_numpy(hit).to(DEV)
    dirty = torch.from_numpy(bad).to(DEV)
    for split in (1, 3, 0):
        want = attention.decode_attention(q, cache, *tabs, split_kv=split)
        got = attention.decode_attention(q, dirty, *tabs, split_kv=split)
        assert bool(torch.isnan(got[hit]).all()), split
        assert torch.equal(got[~hit], want[~hit]), split
    want = attention.decode_attention(q, cache, *tabs, split_kv=2, window=1)
    got = attention.decode_attention(q, dirty, *tabs, split_kv=2, window=1)
    assert torch.equal(got[1:], want[1:])
