"""The 4-bit (OCP MXFP4) paged cache: its format and rounding, the write and read by slot, the append,
and decode attention over it, against the float64 oracle (oracle/kv4.py).

Tolerances. Stored values are compared exactly where nothing is computed (V, unrotated K); a rotated
element may take the neighbouring code where its exact value lies within fp32's error of the border
between them (float64's since the rotation is in double: the last test). Attention: scores are exact
sums over q's E2M3 parts, which hold elements down to 2^-7 (bf16) or 2^-9 (fp16) of their block's largest
whole and cut smaller ones by at most 2^-15 of it; for the normal rows here, where one element in 60 is
that small, and with fp32's sums over a row, that is below 2^-14 of sum |q_i k_i| * scale; a weight is off by that, by the 2^-16 of its two bf16 parts and by fp32; so an output moves
by at most twice the weights' error times (max |v| + |out|), and is rounded once, by half a step of its
type."""
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
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a step


# ---------------------------------------------------------------- the oracle itself (CPU)

def test_oracle_rounds_to_the_nearest_code_and_ties_to_the_even_one():
    row = np.zeros(32)
    row[:9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]
    want = np.zeros(32)
    want[:9] = [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -4.0]
    assert np.array_equal(kv4.held(row), want)
    for top, scale in ((6.9, 127), (7.0, 128), (3.5, 127), (3.49, 126), (1.0, 125)):
        assert kv4.quantize(np.r_[top, np.zeros(31)])[1] == scale
    assert kv4.quantize(np.r_[np.inf, np.zeros(31)])[1] == 255
    assert np.isnan(kv4.held(np.r_[np.nan, np.ones(31)])).all()
    # every representable value is held as it is
    row = np.r_[np.tile(kv4.E2M1, 2), np.tile(-kv4.E2M1, 2)] * 2.0 ** -9
    assert np.array_equal(kv4.held(row), row)


def test_oracle_attention_agrees_with_torch():
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal(s) for s in ((5, 4, 64), (9, 2, 64), (9, 2, 64)))
    seen = np.tril(np.ones((5, 9), bool), 4)
    want = torch.nn.functional.scaled_dot_product_attention(
        *(torch.from_numpy(x).transpose(0, 1) for x in (q, k, v)), attn_mask=torch.from_numpy(seen),
        enable_gqa=True).transpose(0, 1).numpy()
    np.testing.assert_allclose(kv4.attend(q, k, v, seen)[0], want, rtol=0, atol=1e-14)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_oracle_pack_and_unpack_are_inverse(d):
    r = np.random.default_rng(d)
    k, v = (r.standard_normal((2, 3, 16, d)) for _ in range(2))
    cache = kv4.pack(k, v)
    assert cache.shape == (2, 3, layout.KV4_BYTES_PER_DIM * d)
    got = kv4.unpack(cache, d)
    assert np.array_equal(got[0], kv4.held(k)) and np.array_equal(got[1], kv4.held(v))


# ---------------------------------------------------------------- refusals (CPU)

def test_alloc_and_head_dim():
    c = layout.alloc_kv4_cache(5, 2, 128, device="cpu")
    assert c.shape == (5, 2, 2176) and c.dtype == torch.uint8 and not c.any()
    assert layout.is_kv4(c) and layout.kv4_head_dim(c) == 128
    assert layout.kv4_head_dim(c[:, 1:]) == 128
    with pytest.raises(layout.LayoutError):
        layout.alloc_kv4_cache(5, 2, 96, device="cpu")
    for bad in (c[:, :, :100], c[:, :, ::2], c.float(), c[0]):
        with pytest.raises(layout.LayoutError):
            layout.kv4_head_dim(bad)


def _write_args(**kw):
    n, h, d = 3, 2, 64
    a = dict(k_new=torch.zeros(n, h, d, dtype=torch.float16),
             v_new=torch.zeros(n, h, d, dtype=torch.float16),
             cache=layout.alloc_kv4_cache(4, h, d, device="cpu"),
             slots=torch.zeros(n, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(k_new=torch.zeros(3, 2, 64)), dict(v_new=torch.zeros(3, 2, 64)),
    dict(v_new=torch.zeros(2, 2, 64, dtype=torch.float16)),
    dict(k_new=torch.zeros(3, 1, 64, dtype=torch.float16), v_new=torch.zeros(3, 1, 64, dtype=torch.float16)),
    dict(k_new=torch.zeros(3, 64, 2, dtype=torch.float16).transpose(1, 2)),
    dict(cache=torch.zeros(4, 2, 1000, dtype=torch.uint8)),
    dict(cache=torch.zeros(4, 2, 2, 64, dtype=torch.uint8)),
    dict(slots=torch.zeros(2, dtype=torch.int32)), dict(slots=torch.zeros(3)),
    dict(slots=torch.zeros(3, 1, dtype=torch.int32)),
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)),
    dict(inv_freq=torch.zeros(32)), dict(inv_freq=torch.zeros(31), positions=torch.zeros(3, dtype=torch.int32)),
    dict(inv_freq=torch.zeros(32), positions=torch.zeros(3)),
    dict(rope_style=2), dict()])       # the last: all well but for the device
def test_write_refuses(kw):
    with pytest.raises(DecodeArgumentError):
        paging.write_kv4(**_write_args(**kw))


def test_write_and_read_refuse_what_is_no_tensor():
    with pytest.raises(TypeError):
        paging.write_kv4(**_write_args(k_new=[1.0]))
    with pytest.raises(TypeError):
        paging.write_kv4(**_write_args(slots=[0, 1, 2]))
    c = layout.alloc_kv4_cache(4, 2, 64, device="cpu")
    for kw in (dict(dtype=torch.float32), dict(slots=torch.zeros(2)), dict(cache=c[0]), dict()):
        with pytest.raises(DecodeArgumentError):
            paging.read_kv4(**dict(dict(cache=c, slots=torch.zeros(2, dtype=torch.int64)), **kw))


def test_append_refuses():
    a = _write_args()
    ip, ix, ll = (torch.zeros(n, dtype=torch.int32) for n in (4, 3, 3))
    for kw in (dict(k_scale=0.5), dict(kv_indptr=ip[:2]), dict(kv_last_page_len=ll.long()), dict()):
        args = dict(q=None, k_new=a["k_new"], v_new=a["v_new"], kv_data=a["cache"], kv_indptr=ip,
                    kv_indices=ix, kv_last_page_len=ll)
        with pytest.raises(DecodeArgumentError):
            paging.append_kv(**dict(args, **kw))


def _abi(q=0x10000, kv=0x20000, strides=None, opts=None, split=4, d=128, hq=32, hkv=8):
    st = strides or dk_lib.DkStrides(32 * 128, 128, 8 * 2176, 0, 0, 2176, 32 * 128, 128)
    return dk_lib.load().dk_decode_attention_ex(
        q, kv, 0x30000, 0x40000, 0x50000, 0x60000, 0x70000, 1 << 30, 2, hq, hkv, d, 16, 64, 64,
        dk_lib.DK_F16, ctypes.byref(st), split,
        ctypes.byref(opts or dk_lib.options(kv_dtype=dk_lib.DK_KV_MXFP4)), None)


@pytest.mark.parametrize("kw,code", [
    (dict(opts=dict(k_scale=0.5)), dk_lib.DK_EINVAL),
    (dict(opts=dict(qk_path=2)), dk_lib.DK_EINVAL),
    (dict(opts=dict(waves_per_group=2)), dk_lib.DK_EINVAL),
    (dict(kv=0x20008), dk_lib.DK_EUNSUPPORTED),
    (dict(strides=dk_lib.DkStrides(32 * 128, 128, 8 * 2176 + 8, 0, 0, 2176, 32 * 128, 128)),
     dk_lib.DK_EUNSUPPORTED),
    (dict(strides=dk_lib.DkStrides(32 * 128, 128, 8 * 2176, 0, 0, 2177, 32 * 128, 128)),
     dk_lib.DK_EUNSUPPORTED),
    (dict(strides=dk_lib.DkStrides(32 * 128, 128, 8 * 2176, 0, 0, 1 << 29, 32 * 128, 128)),
     dk_lib.DK_EUNSUPPORTED),
    (dict(strides=dk_lib.DkStrides(32 * 128, 128, -16, 0, 0, 2176, 32 * 128, 128)), dk_lib.DK_EINVAL)])
def test_decode_abi_refuses(kw, code):
    if "opts" in kw:
        kw = dict(kw, opts=dk_lib.options(kv_dtype=dk_lib.DK_KV_MXFP4, **kw["opts"]))
    assert _abi(**kw) == code


def test_partials_and_separate_caches_are_refused():
    lib, o = dk_lib.load(), dk_lib.options(kv_dtype=dk_lib.DK_KV_MXFP4)
    st = dk_lib.DkStrides(32 * 128, 128, 8 * 2176, 0, 0, 2176, 32 * 128, 128)
    tail = (0x30000, 0x40000, 0x50000)
    shape = (2, 32, 8, 128, 16, 64, 64, dk_lib.DK_F16, ctypes.byref(st), 4, ctypes.byref(o), None)
    assert lib.dk_decode_partials(0x10000, 0x20000, *tail, 0x70000, 1 << 30, *shape) == \
        dk_lib.DK_EUNSUPPORTED
    assert lib.dk_decode_attention_kv(0x10000, 0x20000, 0x80000, *tail, 0x60000, 0x70000, 1 << 30,
                                      *shape) == dk_lib.DK_EUNSUPPORTED


@pytest.mark.parametrize("args,code", [
    (dict(d=96), dk_lib.DK_EINVAL), (dict(dtype=5), dk_lib.DK_EINVAL), (dict(style=3), dk_lib.DK_EINVAL),
    (dict(slots=None), dk_lib.DK_ENULL), (dict(pos=None, freq=0x1000), dk_lib.DK_ENULL),
    (dict(k=None), dk_lib.DK_ENULL), (dict(cache=0x20004), dk_lib.DK_EUNSUPPORTED),
    (dict(k=0x10008), dk_lib.DK_EUNSUPPORTED), (dict(new_h=60), dk_lib.DK_EUNSUPPORTED),
    (dict(n=-1), dk_lib.DK_EINVAL), (dict(n=0), dk_lib.DK_OK)])
def test_write_abi_refuses(args, code):
    a = dict(k=0x10000, cache=0x20000, slots=0x30000, pos=0x40000, freq=None, style=0, n=3, d=64,
             dtype=0, new_h=64)
    a.update(args)
    st = dk_lib.DkStrides(0, 0, 2 * 1088, 0, 0, 1088, 0, 0)
    assert dk_lib.load().dk_kv4_write(
        None, a["k"], 0x50000, 128, a["new_h"], a["cache"], a["slots"], 0, a["pos"], 0, a["freq"],
        a["style"], a["n"], 1, 2, a["d"], 4, a["dtype"], ctypes.byref(st), None) == code


# ---------------------------------------------------------------- write, read, append (GPU)

def _close_to_held(got, x):
    """Stored values `got` are those held for the exact rows x, or, where x lies at a border within
    fp32's error, the code (or the block's scale) on its other side."""
    want = kv4.held(x)
    x = np.asarray(x, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    top = np.abs(x).reshape(-1, 32).max(1, keepdims=True)
    slack = np.broadcast_to(top * 2.0 ** -20, (top.shape[0], 32)).reshape(x.shape)
    near = np.abs(np.abs(got - x) - np.abs(want - x)) <= slack
    f = np.frexp(top)[0]
    edge = np.broadcast_to(np.abs(f - 0.875) < 2.0 ** -20, (top.shape[0], 32)).reshape(x.shape)
    assert (same | near | edge).all()
    assert (~same).mean() <= 2e-3           # a border within 2^-20 of the block's largest is rare


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_write_holds_every_value_and_tie_and_leaves_the_rest(dtype, d):
    print(f"[case] write {dtype} {d}", flush=True)
    hkv, pages, n = 3, 5, 23
    r = np.random.default_rng(d)
    # all codes, all midpoints, values past 6, tiny and huge blocks, zeros, a NaN and an infinity
    pool = np.r_[kv4.E2M1, (kv4.E2M1[1:] + kv4.E2M1[:-1]) / 2, 6.5, 6.96875, 7.0, 7.5]
    x = r.choice(np.r_[pool, -pool], (2, n, hkv, d)) * 2.0 ** r.integers(-9, 9, (2, n, hkv, 1))
    x[0, 3], x[1, 4] = 0.0, 0.0
    x[0, 5, 0, 1], x[1, 6, 2, 40] = np.nan, -np.inf
    x[0, 7] = r.standard_normal((hkv, d)) * 2.0 ** -20
    kn, vn = (torch.from_numpy(y).to(dtype).to(DEV) for y in x)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    cache = torch.randint(0, 256, (pages, hkv, 17 * d), generator=g, device=DEV, dtype=torch.uint8)
    before = to_np(cache)
    slots = torch.randperm(pages * 16, generator=g, device=DEV)[:n].to(torch.int32)
    slots[10], slots[11] = -1, pages * 16                # no such slot: nothing is written
    paging.write_kv4(kn, vn, cache, slots)
    k, v = paging.read_kv4(cache, slots, torch.bfloat16)
    torch.cuda.synchronize()
    after, at = to_np(cache), to_np(slots)
    with np.errstate(invalid="ignore"):
        uk, uv = kv4.unpack(after, d)
    live = [i for i in range(n) if i not in (10, 11)]
    for t in live:
        p, s = divmod(int(at[t]), 16)
        for got, want in ((uk[p, :, s], kn[t]), (uv[p, :, s], vn[t])):
            np.testing.assert_array_equal(got, kv4.held(to_np(want.double())))
        np.testing.assert_array_equal(to_np(k[t]), uk[p, :, s].astype(np.float32))
        np.testing.assert_array_equal(to_np(v[t]), uv[p, :, s].astype(np.float32))
    assert not to_np(k[10]).any() and not to_np(v[11]).any()
    # every other token's bytes are as they were
    kp, vp, sp = kv4._places(d)
    touched = np.zeros((pages, 17 * d), bool)
    for t in live:
        p, s = divmod(int(at[t]), 16)
        for bytes_ in (kp[0, s], vp[0, s], sp[s], sp[s] + d // 2):
            touched[p, bytes_] = True
    np.testing.assert_array_equal(np.where(touched[:, None], 0, after),
                                  np.where(touched[:, None], 0, before))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,style,n", [
    (torch.float16, 64, 0, 1), (torch.bfloat16, 128, 0, 33), (torch.float16, 256, 1, 17),
    (torch.bfloat16, 64, 1, 200), (torch.float16, 128, 0, 4099)])
def test_write_rotates_like_the_oracle_at_far_positions(dtype, d, style, n):
    print(f"[case] rope {dtype} {d} {style} {n}", flush=True)
    hq, hkv = 5, 2
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    # q a strided view, k and v views of one projection, slots and positions in int64
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device=DEV).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    q0, k0, v0 = (to_np(x.double()) for x in (q, k, v))
    pages = (n + 15) // 16 + 2
    cache = layout.alloc_kv4_cache(pages, hkv, d, device=DEV)
    slots = torch.randperm(pages * 16, generator=g, device=DEV)[:n]
    pos = torch.randint(0, 131072, (n,), generator=g, device=DEV)
    inv = paging.rope_inv_freq(d, theta=500000.0)
    paging.write_kv4(k, v, cache, slots, q=q, inv_freq=inv, positions=pos, rope_style=style)
    kk, vv = paging.read_kv4(cache, slots)
    torch.cuda.synchronize()
    want = kv4.rope(q0, to_np(pos), to_np(inv), style)
    # one rounding, and fp32's error of a rotation (2^-22 of the pair's size)
    np.testing.assert_allclose(to_np(q.double()), want, rtol=EPS[dtype], atol=2.0 ** -20)
    _close_to_held(to_np(kk.double()), kv4.rope(k0, to_np(pos), to_np(inv), style))
    np.testing.assert_array_equal(to_np(vv.double()), kv4.held(v0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,style", [(torch.bfloat16, 64, 0), (torch.float16, 128, 1),
                                           (torch.float16, 256, 0)])
def test_append_writes_each_sequences_last_token(dtype, d, style):
    hq, hkv, lens = 4, 2, [1, 16, 0, 17, 300]
    q, _, ip, ix, ll, _ = layout.synthesize_paged(len(lens), lens, hq, hkv, d, dtype=dtype, device=DEV,
                                                  page_table="permuted", pool_pages=40, seed=d)
    g = torch.Generator(device=DEV)
    g.manual_seed(d)
    k, v = torch.randn(2, len(lens), hkv, d, generator=g, device=DEV).to(dtype).unbind(0)
    inv = paging.rope_inv_freq(d)
    cache = layout.alloc_kv4_cache(40, hkv, d, device=DEV)
    q0 = to_np(q.double())
    paging.append_kv(q, k, v, cache, ip, ix, ll, inv_freq=inv, rope_style=style)
    torch.cuda.synchronize()
    pos = np.array([n - 1 for n in lens])
    wq = kv4.rope(q0, pos, to_np(inv), style)
    wq[2] = q0[2]                                        # no pages: left as it is
    np.testing.assert_allclose(to_np(q.double()), wq, rtol=EPS[dtype], atol=2.0 ** -20)
    uk, uv = kv4.unpack(to_np(cache), d)
    wk = kv4.rope(to_np(k.double()), pos, to_np(inv), style)
    count = 0
    for b, n in enumerate(lens):
        if n:
            p, s = int(ix[ip[b + 1] - 1]), (n - 1) % 16
            _close_to_held(uk[p, :, s], wk[b])
            np.testing.assert_array_equal(uv[p, :, s], kv4.held(to_np(v[b].double())))
            count += hkv * 2
    assert (to_np(cache)[:, :, 16 * d:17 * d] != 0).sum() == count * d // 32   # scales written


# ---------------------------------------------------------------- decode (GPU)

def _filled(pages, hkv, d, seed, gain=1.0):
    """A cache of pages quantised from normal K (some channels stronger) and V, and its bytes."""
    r = np.random.default_rng(seed)
    k = r.standard_normal((pages, hkv, 16, d)) * np.exp(0.6 * r.standard_normal((1, hkv, 1, d))) * gain
    v = r.standard_normal((pages, hkv, 16, d))
    raw = kv4.pack(k.astype(np.float32), v.astype(np.float32))
    return torch.from_numpy(raw).to(DEV), raw


def _decode_case(lens, hq, hkv, d, dtype, seed=0, gain=1.0):
    r = np.random.default_rng(seed)
    np_ = [-(-n // 16) for n in lens]
    pool = sum(np_) + 3
    cache, raw = _filled(pool, hkv, d, seed, gain)
    ids = r.permutation(pool)[:sum(np_)].astype(np.int32)
    ip = np.r_[0, np.cumsum(np_)].astype(np.int32)
    last = np.array([n - 16 * (p - 1) if p else 0 for n, p in zip(lens, np_)], np.int32)
    q = torch.from_numpy(r.standard_normal((len(lens), hq, d))).to(dtype).to(DEV)
    return q, cache, raw, ip, ids, last


def _check(out, q, raw, ip, ids, last, dtype, **kw):
    want, size, big = kv4.decode(to_np(q.double()), raw, ip, ids, last, **kw)
    weight = 2 * (size * 2.0 ** -14 + 2.0 ** -15)
    tol = EPS[dtype] * np.abs(want) * (1 + weight) + weight * (big + np.abs(want)) + 2.0 ** -25
    got = to_np(out.double())
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / tol
    assert worst.max(initial=0) <= 1.0, worst.max()
    # over all outputs the errors do not add up: the norm's error is that of the rounding
    norm = np.linalg.norm(want)
    if want.size >= 4096 and norm:
        exact = np.linalg.norm(to_np(torch.from_numpy(want).to(dtype).double()) - want) / norm
        assert np.linalg.norm(got - want) / norm <= 1.2 * exact + size * 2.0 ** -17


CASES = [
    # lens, hq, hkv, d
    ([1], 1, 1, 128), ([2, 16, 17, 15, 0, 64, 65], 8, 2, 64), ([1, 0, 33], 8, 8, 256),
    ([300, 5, 1111], 32, 8, 128), ([47, 48, 49], 20, 4, 128), ([100, 700], 16, 2, 64),
    ([513], 40, 8, 64), ([129, 64, 63], 32, 2, 128), ([77, 500], 48, 3, 256), ([260], 17, 1, 256),
    ([90], 80, 2, 128), ([3, 200], 33, 1, 64), ([31, 1500], 6, 6, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,hq,hkv,d", CASES)
def test_decode_matches_the_oracle_in_every_schedule(lens, hq, hkv, d, dtype):
    q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, dtype, seed=hq + d)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    for kw in (dict(split_kv=1), dict(split_kv=3), dict(split_kv=0),
               dict(split_kv=0, max_pages_per_seq=attention.plan_hint(ip)),
               dict(split_kv=0, schedule=1, waves_per_cu=1), dict(split_kv=0, schedule=2)):
        print(f"[case] decode {lens} {hq}/{hkv}/{d} {dtype} {kw}", flush=True)
        out = attention.decode_attention(q, cache, *tabs, **kw)
        torch.cuda.synchronize()
        _check(out, q, raw, ip, ids, last, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hq,hkv", [(64, 16, 2), (128, 8, 2), (256, 16, 1)])
@pytest.mark.parametrize("opt", [dict(window=1), dict(window=100), dict(logit_cap=20.0),
                                 dict(sinks=True), dict(sm_scale=0.3),
                                 dict(window=37, logit_cap=5.0, sinks=True)])
def test_decode_options(opt, d, hq, hkv, dtype):
    lens = [1, 36, 37, 38, 200, 0, 777]
    q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, dtype, seed=d)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    kw, okw = dict(opt), {}
    if "sinks" in kw:
        kw["sinks"] = torch.linspace(-2, 3, hq, device=DEV)
        okw["sinks"] = to_np(kw["sinks"].double())
    okw.update(window=opt.get("window", 0), cap=opt.get("logit_cap", 0.0), scale=opt.get("sm_scale"))
    for split in (1, 2, 0):
        print(f"[case] options {opt} {d} {dtype} split {split}", flush=True)
        out = attention.decode_attention(q, cache, *tabs, split_kv=split, **kw)
        torch.cuda.synchronize()
        _check(out, q, raw, ip, ids, last, dtype, **okw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_of_a_dominant_key_keeps_the_others(dtype):
    # one key far above 500 others, its V zero: the output is the others' small weights alone
    d, n = 128, 501
    r = np.random.default_rng(3)
    k = r.standard_normal((32, 1, 16, d)) * 0.1
    v = r.standard_normal((32, 1, 16, d))
    q = r.standard_normal((1, 4, d))
    q[:, :] = q[:, :1]
    k[0, 0, 0] = q[0, 0] * 1.35
    v[0, 0, 0] = 0.0
    raw = kv4.pack(k, v)
    qt = torch.from_numpy(q).to(dtype).to(DEV)
    ip, ids, last = np.array([0, 32], np.int32), np.arange(32, dtype=np.int32), np.array([5], np.int32)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    out = attention.decode_attention(qt, torch.from_numpy(raw).to(DEV), *tabs, split_kv=1)
    want, size, _ = kv4.decode(to_np(qt.double()), raw, ip, ids, last)
    # relative to the output: weights of the others are exact to 2^-16 whatever the dominant one's
    got = to_np(out.double())
    assert np.abs(want).max() < 1e-2 and n == 16 * 31 + 5
    step = 2.0 ** -25 if dtype == torch.float16 else 0.0     # fp16's subnormal half step
    assert np.linalg.norm(got - want) <= (EPS[dtype] + size * 2.0 ** -14) * np.linalg.norm(want) + \
        step * np.sqrt(want.size)


@pytest.mark.gpu
def test_decode_ignores_what_lies_behind_the_last_token_and_before_the_window():
    # bytes of tokens that are not attended to hold every pattern, NaN scales among them
    lens, hq, hkv, d = [5, 40, 130], 8, 2, 128
    for dtype in (torch.float16, torch.bfloat16):
        q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, dtype, seed=9)
        tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
        bad = raw.copy()
        kp, vp, sp = kv4._places(d)
        live = {int(ids[ip[b] + t // 16]) * 16 + t % 16 for b, n in enumerate(lens)
                for t in range(max(0, n - 50), n)}
        for p in range(bad.shape[0]):
            for s in range(16):
                if 16 * p + s not in live:
                    for bytes_ in (sp[s], sp[s] + d // 2):
                        bad[p][:, bytes_] = 255
                    bad[p][:, kp[0, s]] = 0x77
                    bad[p][:, vp[0, s]] = 0xff
        dirty = torch.from_numpy(bad).to(DEV)
        for kw in (dict(split_kv=1, window=50), dict(split_kv=2, window=50), dict(split_kv=0, window=50)):
            a = attention.decode_attention(q, cache, *tabs, **kw)
            b = attention.decode_attention(q, dirty, *tabs, **kw)
            assert torch.equal(a, b)
        # and a NaN that is attended to shows, in its sequence and kv head alone
        bad = raw.copy()
        p = int(ids[ip[1]])
        bad[p, 1, sp[3, 0]] = 255
        for kw in (dict(split_kv=1), dict(split_kv=2), dict(split_kv=0)):
            out = to_np(attention.decode_attention(q, torch.from_numpy(bad).to(DEV), *tabs, **kw).float())
            assert np.isnan(out[1, 4:]).all()
            assert np.isfinite(out[1, :4]).all() and np.isfinite(out[[0, 2]]).all()


@pytest.mark.gpu
def test_decode_strided_views_outputs_workspaces_and_plans():
    lens, hq, hkv, d = [70, 300], 8, 4, 128
    q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, torch.bfloat16, seed=4)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    want = attention.decode_attention(q, cache, *tabs, split_kv=2)
    # a slice of kv heads, every other page of a larger pool, q and out as views, odd out rows
    big = torch.zeros(2 * cache.shape[0], hkv + 1, 17 * d + 16, dtype=torch.uint8, device=DEV)
    view = big[::2, 1:, :17 * d]
    view.copy_(cache)
    buf = torch.zeros(2, hq, d + 1, dtype=torch.bfloat16, device=DEV)
    for split in (1, 2, 0):
        one = attention.decode_attention(q, cache, *tabs, split_kv=split)
        assert torch.equal(attention.decode_attention(q, view, *tabs, split_kv=split), one)
        out = attention.decode_attention(q, view, *tabs, split_kv=split, out=buf[:, :, :d])
        assert out.data_ptr() == buf.data_ptr() and torch.equal(out, one)
    assert not buf[:, :, d].any()
    half = attention.decode_attention(q[:, 4:], cache[:, 2:], *tabs, split_kv=2)
    assert torch.equal(half, want[:, 4:])
    plan = attention.DecodePlan(q, cache, *tabs, split_kv=2)
    assert torch.equal(plan.run(q, cache, *tabs), want)
    with pytest.raises(DecodeArgumentError):
        plan.run(q, cache[:, :2], *tabs)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=DEV).fill_(255)
    assert torch.equal(plan.run(q, cache, *tabs, workspace=ws), want)
    with pytest.raises(DecodeArgumentError):
        attention.decode_attention(q, cache, *tabs, k_scale=0.5)
    with pytest.raises(DecodeArgumentError):
        attention.decode_partials(q, cache, *tabs, 2)
    with pytest.raises(DecodeArgumentError):
        attention.decode_attention(q, cache[:, :, :1088], *tabs)


@pytest.mark.gpu
def test_decode_captured_and_replayed_beside_eager_work():
    lens, hq, hkv, d = [90, 700, 33], 8, 2, 64
    q, cache, raw, ip, ids, last = _decode_case(lens, hq, hkv, d, torch.float16, seed=6)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    side = torch.cuda.Stream()
    graphs = []
    for split in (2, 0):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            attention.decode_attention(q, cache, *tabs, split_kv=split)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attention.decode_attention(q, cache, *tabs, split_kv=split)
        graphs.append((g, out, split))
    for step in range(4):
        q.copy_(torch.randn_like(q))
        for g, out, split in graphs:
            g.replay()
            want = attention.decode_attention(q, cache, *tabs, split_kv=split)
            torch.cuda.synchronize()
            assert torch.equal(out, want), (step, split)


@pytest.mark.gpu
def test_decode_offsets_past_32_bits():
    # pages whose bytes start beyond 2^32: a pool of 5 GiB, three live pages in its last part
    d, hkv, hq = 128, 8, 32
    pages = (5 << 30) // (hkv * 17 * d)
    cache = torch.zeros(pages, hkv, 17 * d, dtype=torch.uint8, device=DEV)
    part, raw = _filled(3, hkv, d, 8)
    ids = np.array([pages - 1, pages // 2 + 7, pages - 100], np.int32)
    cache[torch.from_numpy(ids).long().to(DEV)] = part
    r = np.random.default_rng(8)
    q = torch.from_numpy(r.standard_normal((1, hq, d))).half().to(DEV)
    ip, last = np.array([0, 3], np.int32), np.array([9], np.int32)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    for split in (1, 3, 0):
        out = attention.decode_attention(q, cache, *tabs, split_kv=split)
        torch.cuda.synchronize()
        _check(out, q, raw, ip, np.arange(3, dtype=np.int32), last, torch.float16)
    # write and read there too
    slots = torch.tensor([int(ids[0]) * 16 + 15, int(ids[1]) * 16], device=DEV)
    k, v = torch.randn(2, 2, hkv, d, device=DEV).half().unbind(0)
    paging.write_kv4(k, v, cache, slots)
    kk, vv = paging.read_kv4(cache, slots)
    np.testing.assert_array_equal(to_np(kk.double()), kv4.held(to_np(k.double())))
    np.testing.assert_array_equal(to_np(vv.double()), kv4.held(to_np(v.double())))


@pytest.mark.gpu
def test_decode_bad_page_ids_stay_inside_the_pool():
    # ids outside the pool read page 0, as over the other caches
    q, cache, raw, ip, ids, last = _decode_case([40, 20], 4, 2, 64, torch.float16, seed=2)
    tabs = [torch.from_numpy(x).to(DEV) for x in (ip, ids, last)]
    bad, zero = tabs[1].clone(), tabs[1].clone()
    bad[0], bad[2] = 2 ** 31 - 1, -5
    zero[0], zero[2] = 0, 0
    for split in (1, 2, 0):
        assert torch.equal(attention.decode_attention(q, cache, tabs[0], bad, tabs[2], split_kv=split),
                           attention.decode_attention(q, cache, tabs[0], zero, tabs[2], split_kv=split))


@pytest.mark.gpu
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rotated_codes_are_those_of_the_exact_rotation(dtype, style):
    """Each code is the one that the rotation in 64 bits rounds to, also beside a boundary between two
    codes: of 17 million elements an fp32 rotation puts about two on the other side. The 64-bit result
    is itself off by 2^-52 or so, which reaches a boundary with a chance of 1e-8."""
    n, hkv, d = 16384, 8, 128
    g = torch.Generator().manual_seed(11 + style)
    k = torch.randn(n, hkv, d, generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, 131072, (n,), generator=g, dtype=torch.int32)
    pos[:5] = torch.tensor([0, 1, 2, 131071, 0])
    pos = pos.to(DEV)
    inv = paging.rope_inv_freq(d, theta=500000.0)
    cache = layout.alloc_kv4_cache(n // 16, hkv, d, device=DEV)
    slots = torch.arange(n, device=DEV)
    paging.write_kv4(k, k, cache, slots, inv_freq=inv, positions=pos, rope_style=style)
    got = paging.read_kv4(cache, slots)[0].double()
    angle = pos.double()[:, None] * inv.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x = k.double()
    lo, hi = (slice(0, d // 2), slice(d // 2, d)) if style == 0 else (slice(0, d, 2), slice(1, d, 2))
    y = torch.empty_like(x)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    b = y.reshape(-1, 32)
    man, ex = torch.frexp(b.abs().amax(1, keepdim=True))      # man in [1/2, 1)
    unit = torch.exp2((ex - 3 + (man >= 0.875).to(ex.dtype)).double())
    z = b / unit
    step = torch.where(z.abs() < 2, 0.5, torch.where(z.abs() < 4, 1.0, 2.0))
    want = ((z / step).round() * step * unit).reshape(y.shape)
    assert int((got != want).sum()) == 0


@pytest.mark.parametrize("q_strides,cache_strides", [
    ((128, 0), (2176, 1088)), ((64, 64), (2176, 1088)), ((0, 64), (2176, 1088)),
    ((128, 64), (0, 1088)), ((128, 64), (2176, 1072))])
def test_write_refuses_rows_that_overlap(q_strides, cache_strides):
    st = dk_lib.DkStrides(*q_strides, cache_strides[0], 0, 0, cache_strides[1], 0, 0)
    lib = dk_lib.load()
    assert lib.dk_kv4_write(0x60000, 0x10000, 0x50000, 128, 64, 0x20000, 0x30000, 0, 0x40000, 0, 0x70000, 0, 3, 2,
                            2, 64, 4, 0, ctypes.byref(st), None) == dk_lib.DK_EUNSUPPORTED
    assert b"overlap" in lib.dk_last_error()


def test_read_refuses_rows_that_overlap():
    for out_t, out_h in ((128, 0), (64, 64), (0, 64)):
        assert dk_lib.load().dk_kv4_read(0x20000, 2176, 1088, 0x30000, 0, 0x40000, 0x50000, out_t, out_h, 3, 2,
                                         64, 4, 0, None) == dk_lib.DK_EUNSUPPORTED
