"""Prefill attention over the 4-bit cache (extend.extend_attention_kv4) against the float64 oracle
(oracle/kv4.py), its refusals, and chunked prefill followed by decode.

Tolerance: the scores are fp32 sums of exact products over q's three E2M3 parts: off by at most 2^-17 of
sum |q_i k_i| * scale (128 additions of half a step of 2^-24, and the rounding of the softmax scale), and by
what the parts leave of q, at most 2^-15 of the power of two below a block's largest magnitude, of
elements below 2^-4 (fp16) or 2^-7 (bf16) of it. In normal rows the largest of 32 lies below 4, that power
is at most 2, and one element in 10 is below an eighth: their share, 0.1 * 2 * 2^-15 |k|, is 2^-17 of the
mean 0.8 |k| of all; so 2^-16 in fp16, and 2^-17 with a twentieth of it more in bf16; a weight enters as two parts of q's type: the first leaves at most half a step, 2^-11
of it in fp16 and 2^-8 in bf16, the second as much of that, so 2^-22 and 2^-16 of the weight (in fp16 never
finer than 2^-24 of the largest); one rounding of the output."""
import ctypes

import numpy as np
import pytest
import torch

import attention
import dk_lib
import extend
import layout
import paging
from dk_lib import DecodeArgumentError
from helpers import to_np
from oracle import kv4

DEV = "cuda"
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _args(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.float16), cache=layout.alloc_kv4_cache(4, 2, 64, device="cpu"),
             block_table=torch.zeros(2, 4, dtype=torch.int32), rows=[0], new_lens=[3], all_lens=[3])
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 3, 64, dtype=torch.float16)),
    dict(q=torch.zeros(3, 4, 128, dtype=torch.float16)), dict(q=torch.zeros(3, 64, 4, dtype=torch.float16).transpose(1, 2)),
    dict(cache=torch.zeros(4, 2, 100, dtype=torch.uint8)), dict(cache=torch.zeros(4, 2, 64, dtype=torch.float16)),
    dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), dict(block_table=torch.zeros(8, dtype=torch.int32)),
    dict(new_lens=[1, 2]), dict(all_lens=[2 ** 40]), dict(out=torch.zeros(3, 4, 64)), dict(scale=-1.0),
    dict(scale=float("nan")), dict(logit_cap=-1.0), dict(window=-1), dict(window=2.0),
    dict(sinks=torch.zeros(3)), dict()])          # the last: all well but for the device
def test_refusals(kw):
    with pytest.raises(DecodeArgumentError):
        extend.extend_attention_kv4(**_args(**kw))


@pytest.mark.parametrize("kw,code", [
    (dict(rows=[4]), dk_lib.DK_EINVAL), (dict(rows=[-1]), dk_lib.DK_EINVAL),
    (dict(all=[65]), dk_lib.DK_EINVAL), (dict(new=[-1]), dk_lib.DK_EINVAL),
    (dict(new=[4], all=[3]), dk_lib.DK_EINVAL), (dict(new=[8], all=[8]), dk_lib.DK_EINVAL),
    (dict(q=0x10008), dk_lib.DK_EUNSUPPORTED), (dict(cache=0x20008), dk_lib.DK_EUNSUPPORTED),
    (dict(q_h=60), dk_lib.DK_EUNSUPPORTED), (dict(kv_p=2200), dk_lib.DK_EUNSUPPORTED),
    (dict(pages=0), dk_lib.DK_EINVAL), (dict(table=None), dk_lib.DK_ENULL), (dict(d=32), dk_lib.DK_EINVAL),
    (dict(scale=0.0), dk_lib.DK_EINVAL), (dict(blocks=9), dk_lib.DK_EINVAL),
    (dict(o_h=0), dk_lib.DK_EUNSUPPORTED), (dict(o_h=56), dk_lib.DK_EUNSUPPORTED),
    (dict(new=[0], all=[0], q=None), dk_lib.DK_OK)])
def test_abi_refusals(kw, code):
    a = dict(q=0x10000, cache=0x20000, kv_p=2176, table=0x30000, rows=[1], new=[3], all=[3], d=64, pages=8,
             q_h=64, o_h=64, scale=0.1, blocks=4)
    a.update(kw)
    i32 = ctypes.c_int32 * 1
    s = dk_lib.DkExtendStrides(256, a["q_h"], 0, 0, 0, 0, 256, a["o_h"])
    assert dk_lib.load().dk_extend_attention_kv4(
        a["q"], a["cache"], a["kv_p"], 1088, a["table"], 8, 4, a["blocks"], i32(*a["rows"]), i32(*a["new"]),
        i32(*a["all"]), 0x40000, None, 0, 1, 7, 4, 2, a["d"], a["pages"], 0, ctypes.byref(s), a["scale"], 0.0,
        0, None, None) == code


def test_workspace_bytes():
    """Room for the partials of the split that a call takes: none for a short or an empty one, none past
    what the tiles of a full chip take, never more than the largest split's."""
    lib = dk_lib.load()

    def need(new, alls, hq, hkv, d, window=0):
        ints = ctypes.c_int32 * len(new)
        return lib.dk_extend_kv4_workspace_bytes(len(new), ints(*new), ints(*alls), hq, hkv, d, window)

    assert need([0, 0], [5, 0], 8, 2, 64) == need([3], [200], 8, 2, 64) == need([512], [512], 32, 8, 128) == 0
    assert need([2048], [8192], 32, 8, 128) == 0 and need([-1], [5], 8, 2, 64) == 0
    assert need([4], [8000], 8, 2, 64, window=100) == 0
    for d in (64, 128, 256):
        some = need([16], [8000], 32, 8, d)
        ints = ctypes.c_int32 * 1
        assert 0 < some <= lib.dk_extend_workspace_bytes(1, ints(16), ints(8000), 32, 8, d, 0)
        assert some % (16 * 32 * (d + 2) * 4) == 0            # whole rows of O, m and l


def _case(reqs, hq, hkv, d, dtype, seed):
    """reqs: (prefix, new) per request. Pages in random order, unused table entries outside the cache."""
    r = np.random.default_rng(seed)
    alls = [p + n for p, n in reqs]
    blocks = [-(-n // 16) for n in alls]
    pool = sum(blocks) + 2
    k = r.standard_normal((pool, hkv, 16, d)) * np.exp(0.6 * r.standard_normal((1, hkv, 1, d)))
    raw = kv4.pack(k.astype(np.float32), r.standard_normal((pool, hkv, 16, d)).astype(np.float32))
    ids = r.permutation(pool).astype(np.int32)
    table = np.full((len(reqs) + 2, max(blocks) + 1), 2 ** 30, np.int32)
    rows = r.permutation(len(reqs) + 2)[:len(reqs)]
    at = 0
    for row, n in zip(rows, blocks):
        table[row, :n] = ids[at:at + n]
        at += n
    q = torch.from_numpy(r.standard_normal((sum(n for _, n in reqs) + 1, hq, d))).to(dtype).to(DEV)
    return q, torch.from_numpy(raw).to(DEV), raw, table, [int(x) for x in rows], [n for _, n in reqs], alls


def _oracle(q, raw, table, rows, new, alls, window=0, **kw):
    d = q.shape[2]
    with np.errstate(invalid="ignore"):
        kk, vv = kv4.unpack(raw, d)
    out, size, big, at = np.zeros(q.shape), 0.0, 0.0, 0
    for row, n, total in zip(rows, new, alls):
        pages = table[row, :-(-total // 16)]
        k, v = (x[pages].transpose(0, 2, 1, 3).reshape(-1, raw.shape[1], d)[:total] for x in (kk, vv))
        pos = np.arange(total - n, total)[:, None]
        t = np.arange(total)[None]
        seen = t <= pos
        if window:
            seen &= t > pos - window
        out[at:at + n], s = kv4.attend(q[at:at + n], k, v, seen, **kw)
        size, big, at = max(size, s), max(big, float(np.abs(v).max(initial=0))), at + n
    return out, size, big


def _check(got, want, size, big, dtype):
    weight = 2 * (size * 2.0 ** -16 + (2.0 ** -20 if dtype == torch.float16 else 2.0 ** -16))
    tol = EPS[dtype] * np.abs(want) * (1 + weight) + weight * (big + np.abs(want)) + 2.0 ** -23
    worst = np.abs(to_np(got.double()) - want) / tol
    assert worst.max(initial=0) <= 1.0, worst.max()


CASES = [
    ([(0, 1)], 1, 1, 128), ([(0, 40), (3, 1), (100, 33), (5, 0)], 8, 2, 64),
    ([(15, 1), (16, 1), (17, 70), (63, 66)], 4, 4, 128), ([(0, 200), (1, 130)], 16, 2, 256),
    ([(700, 16)], 32, 8, 128), ([(1000, 3), (2, 65)], 5, 1, 64), ([(300, 129)], 6, 2, 128),
    ([(0, 64), (64, 64)], 40, 8, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reqs,hq,hkv,d", CASES)
def test_matches_the_oracle(reqs, hq, hkv, d, dtype):
    q, cache, raw, table, rows, new, alls = _case(reqs, hq, hkv, d, dtype, hq + d)
    t = torch.from_numpy(table).to(DEV)
    for kw in (dict(), dict(window=1), dict(window=50, logit_cap=20.0), dict(sinks=True, scale=0.2)):
        print(f"[case] extend kv4 {reqs} {hq}/{hkv}/{d} {dtype} {kw}", flush=True)
        okw = dict(window=kw.get("window", 0), cap=kw.get("logit_cap", 0.0), scale=kw.get("scale"))
        kw = dict(kw)
        if "sinks" in kw:
            kw["sinks"] = torch.linspace(-2, 3, hq, device=DEV)
            okw["sinks"] = to_np(kw["sinks"].double())
        out = torch.full_like(q, 7.0)
        got = extend.extend_attention_kv4(q, cache, t, rows, new, alls, out=out, **kw)
        torch.cuda.synchronize()
        assert got is out and (out[-1] == 7.0).all()          # the row behind the last new token
        _check(out[:-1], *(_oracle(to_np(q.double())[:-1], raw, table, rows, new, alls, **okw)), dtype)


@pytest.mark.gpu
def test_strided_q_and_out_a_slice_of_heads_and_host_tensors():
    reqs, hq, hkv, d = [(20, 50), (0, 9)], 8, 4, 128
    q, cache, raw, table, rows, new, alls = _case(reqs, hq, hkv, d, torch.float16, 1)
    t = torch.from_numpy(table).to(DEV)
    want = extend.extend_attention_kv4(q, cache, t, rows, new, alls)
    qkv = torch.zeros(q.shape[0], hq + 3, d, dtype=q.dtype, device=DEV)
    qkv[:, 2:2 + hq] = q
    out = torch.zeros(q.shape[0], hq + 1, d, dtype=q.dtype, device=DEV)
    wide = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + table.shape[1]] = t
    extend.extend_attention_kv4(qkv[:, 2:2 + hq], cache, wide[:, 3:3 + table.shape[1]], np.array(rows),
                                torch.tensor(new), tuple(alls), out=out[:, 1:])
    n = sum(new)
    assert torch.equal(out[:n, 1:], want[:n]) and not out[:, 0].any()
    half = extend.extend_attention_kv4(q[:, 4:], cache[:, 2:], t, rows, new, alls)
    assert torch.equal(half[:n], want[:n, 4:])
    with pytest.raises(DecodeArgumentError):
        extend.extend_attention_kv4(q, cache, t, torch.tensor(rows, device=DEV), new, alls)
    with pytest.raises(DecodeArgumentError):
        extend.extend_attention_kv4(q, cache.cpu(), t, rows, new, alls)
    assert extend.extend_attention_kv4(q[:0], cache, t, [], [], []).shape == (0, hq, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_lies_behind_a_request_is_not_read_and_bad_pages_give_nan(d, dtype):
    reqs = [(10, 23), (70, 30)]
    q, cache, raw, table, rows, new, alls = _case(reqs, 4, 2, d, dtype, d)
    t = torch.from_numpy(table).to(DEV)
    want = extend.extend_attention_kv4(q, cache, t, rows, new, alls)
    bad = raw.copy()
    kp, vp, sp = kv4._places(d)
    for row, n in zip(rows, alls):                            # tokens behind the last one
        p = table[row, n // 16]
        for s in range(n % 16, 16):
            bad[p][:, kp[0, s]], bad[p][:, vp[0, s]] = 0x7f, 0xf7
            bad[p][:, sp[s]] = bad[p][:, sp[s] + d // 2] = 255
    got = extend.extend_attention_kv4(q, torch.from_numpy(bad).to(DEV), t, rows, new, alls)
    assert torch.equal(got[:-1], want[:-1])
    # a page outside the cache: NaN for the tokens that attend to it (request 1's tokens from 80 on)
    tb = table.copy()
    tb[rows[1], 5] = -1
    got = extend.extend_attention_kv4(q, cache, torch.from_numpy(tb).to(DEV), rows, new, alls)
    flags = [bool(torch.isnan(x).all()) for x in got[:-1]]
    assert flags == [False] * 23 + [70 + i >= 80 for i in range(30)]
    assert torch.equal(got[:33], want[:33])
    # a NaN block that is attended to
    nanned = raw.copy()
    nanned[table[rows[0], 0], 1, sp[4, 0]] = 255
    got = to_np(extend.extend_attention_kv4(q, torch.from_numpy(nanned).to(DEV), t, rows, new, alls).float())
    assert np.isnan(got[:23, 2:]).all() and np.isfinite(got[:23, :2]).all() and np.isfinite(got[23:-1]).all()


# More query tiles than workgroups that the chip holds per kv head, so that workgroups take several;
# more than a call deals out; more requests than a launch takes
MANY = [
    ([(0, 300), (7, 129), (64, 1), (0, 0), (33, 260), (5, 40), (0, 513)], 64, 64, 64),
    ([(0, 300), (7, 129), (64, 1), (33, 260)], 100, 50, 128), ([(9, 257), (0, 140)], 60, 60, 256),
    ([(0, 140), (3, 129)], 300, 300, 64), ([(i % 50, 1 + i % 3) for i in range(270)], 4, 2, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("reqs,hq,hkv,d", MANY)
def test_many_tiles(reqs, hq, hkv, d):
    q, cache, raw, table, rows, new, alls = _case(reqs, hq, hkv, d, torch.bfloat16, hq)
    t = torch.from_numpy(table).to(DEV)
    for window in (0, 70):
        out = torch.full_like(q, 7.0)
        got = extend.extend_attention_kv4(q, cache, t, rows, new, alls, out=out, window=window or None)
        assert got is out and bool((out[sum(new):] == 7.0).all())
        some, g = sorted({0, hkv // 2, hkv - 1}), hq // hkv    # kv heads, and their q heads
        heads = [x * g + i for x in some for i in range(g)]
        want, size, big = _oracle(to_np(q[:, heads].double()), raw[:, some], table, rows, new, alls, window)
        _check(got[:-1, heads], want[:-1], size, big, torch.bfloat16)
        for _ in range(2):
            again = extend.extend_attention_kv4(q, cache, t, rows, new, alls, window=window or None)
            assert torch.equal(again[:-1], got[:-1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_values_reach_only_those_that_attend_to_them(d, dtype, window):
    """A value block with the NaN scale: the outputs of its dims, for the queries that see its token;
    every other output keeps its bits, though the tile that holds the token is theirs too."""
    reqs = [(10, 123), (90, 60), (0, 7)]
    q, cache, raw, table, rows, new, alls = _case(reqs, 6, 2, d, dtype, d + window)
    t = torch.from_numpy(table).to(DEV)
    kw = dict(window=window or None)
    want = extend.extend_attention_kv4(q, cache, t, rows, new, alls, **kw)
    sp = kv4._places(d)[2]
    nanned = raw.copy()
    hit = np.zeros(tuple(want.shape), bool)
    starts = np.cumsum([0] + new)
    for req, tok, kvh, block in ((0, 3, 0, 0), (0, 60, 1, d // 32 - 1), (0, 100, 1, 0), (1, 95, 0, 1),
                                 (1, 149, 1, 0), (2, 6, 0, 0)):
        nanned[table[rows[req], tok // 16], kvh, sp[tok % 16, block] + d // 2] = 255
        for i in range(new[req]):
            pos = reqs[req][0] + i
            if tok <= pos and (not window or tok > pos - window):
                hit[starts[req] + i, 3 * kvh:3 * kvh + 3, 32 * block:32 * block + 32] = True
    got = extend.extend_attention_kv4(q, torch.from_numpy(nanned).to(DEV), t, rows, new, alls, **kw)
    hit = torch.from_numpy(hit[:-1]).to(DEV)
    assert bool(torch.isnan(got[:-1][hit]).all())
    assert torch.equal(got[:-1][~hit], want[:-1][~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_split_keys_keep_nan(d):
    """Few queries over many keys: the key ranges' partials carry a bad page's and a value's NaN."""
    q, cache, raw, table, rows, new, alls = _case([(2990, 3)], 4, 2, d, torch.bfloat16, d)
    t = torch.from_numpy(table).to(DEV)
    i32 = ctypes.c_int32 * 1
    assert dk_lib.load().dk_extend_kv4_workspace_bytes(1, i32(3), i32(2993), 4, 2, d, 0) > 0
    want = extend.extend_attention_kv4(q, cache, t, rows, new, alls)
    tb = table.copy()
    tb[rows[0], 187] = 2 ** 31 - 1                           # tokens 2992 ..: the last query's alone
    got = extend.extend_attention_kv4(q, cache, torch.from_numpy(tb).to(DEV), rows, new, alls)
    assert torch.equal(got[:2], want[:2]) and bool(torch.isnan(got[2]).all())
    nanned = raw.copy()
    nanned[table[rows[0], 5], 1, kv4._places(d)[2][7, 1] + d // 2] = 255
    got = extend.extend_attention_kv4(q, torch.from_numpy(nanned).to(DEV), t, rows, new, alls)
    assert bool(torch.isnan(got[:3, 2:, 32:64]).all())
    assert torch.equal(got[:3, :2], want[:3, :2]) and torch.equal(got[:3, 2:, :32], want[:3, 2:, :32])
    assert torch.equal(got[:3, 2:, 64:], want[:3, 2:, 64:])


@pytest.mark.gpu
def test_fp16_values_at_the_end_of_its_range():
    # a block of 65,504s is held as 65,536: staged at half its size it stays finite
    d = 64
    k, v = np.zeros((1, 1, 16, d)), np.zeros((1, 1, 16, d))
    k[0, 0, :, :], v[0, 0, 0, :32] = 65504.0, 65504.0
    raw = kv4.pack(k, v)
    q = torch.zeros(4, 1, d, dtype=torch.float16, device=DEV)
    q[:, :, 0] = 2.0 ** -16
    table = np.zeros((1, 1), np.int32)
    got = extend.extend_attention_kv4(q, torch.from_numpy(raw).to(DEV), torch.from_numpy(table).to(DEV), [0], [4],
                                      [4])
    want, *_ = _oracle(to_np(q.double()), raw, table, [0], [4], [4])
    assert want[1, 0, 0] == 32768.0
    np.testing.assert_allclose(to_np(got.double())[1:], want[1:], rtol=2.0 ** -10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,hq,hkv", [(torch.bfloat16, 128, 8, 2), (torch.float16, 64, 6, 2)])
def test_chunked_prefill_then_decode_is_one_history(dtype, d, hq, hkv):
    """Two requests prefilled in chunks through tables, write and prefill attention, then decoded:
    each step against the oracle over the cache as it stands."""
    r = np.random.default_rng(d)
    pool = 30
    cache = layout.alloc_kv4_cache(pool, hkv, d, device=DEV)
    table = torch.full((4, 10), -1, dtype=torch.int32, device=DEV)
    rows, cached = [2, 1], np.zeros(2, int)
    rows_t = torch.tensor(rows, device=DEV)
    free = list(r.permutation(pool))
    inv = paging.rope_inv_freq(d)
    for step, new in enumerate(([40, 17], [9, 0], [70, 16], [1, 1], [1, 1])):
        new = np.array(new)
        alls = cached + new
        need = int((-(-alls // 16) - -(-cached // 16)).sum())
        st = paging.grow_block_tables(
            table, rows_t, torch.from_numpy(cached).to(DEV), torch.from_numpy(new).to(DEV),
            torch.tensor([free.pop() for _ in range(need)], dtype=torch.int32, device=DEV), int(new.sum()),
            int((-(-alls // 16)).sum()))
        q, k, v = (torch.from_numpy(r.standard_normal((int(new.sum()), h, d))).to(dtype).to(DEV)
                   for h in (hq, hkv, hkv))
        paging.write_kv4(k, v, cache, st.slots, q=q, inv_freq=inv, positions=st.positions)
        out = extend.extend_attention_kv4(q, cache, table, rows, new, alls)
        want, size, big = _oracle(to_np(q.double()), to_np(cache), to_np(table), rows, new, alls)
        _check(out, want, size, big, dtype)
        if step >= 3:                                        # a decode step's two paths agree
            dec = attention.decode_attention(q, cache, st.kv_indptr, st.kv_indices, st.kv_last_page_len,
                                             split_kv=0)
            weight = 2 * (size * 2.0 ** -14 + 2.0 ** -15)
            assert (np.abs(to_np(dec.double()) - want) <=
                    EPS[dtype] * np.abs(want) * (1 + weight) + weight * (big + np.abs(want)) + 2.0 ** -25).all()
        cached = alls
