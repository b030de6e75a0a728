"""The paged decoder cache: vtx_kv_append_paged, vtx_flash_attn_paged,
vtx_kv_score_paged and vtx_kv_evict_paged against plain 64-bit forms
(paged_ref.py), their refusals, and a run of them together."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import paged_ref as R
import vtx_attn as V

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
B = ctypes.byref
BASE = 1e6


@pytest.fixture(scope="module")
def lib():
    import build as b
    b.build()
    return V.load()


# ---- the C ABI without a device --------------------------------------------------

def test_paged_struct_layouts(tmp_path):
    probes = {"vtx_paged_kv": (V.VtxPagedKv, ["v", "page_table", "q_start", "max_pages", "max_kv_len"]),
              "vtx_kv_append_paged_args": (V.KvAppendPagedArgs, ["freq_base", "row_cap", "q_out", "positions", "score"]),
              "vtx_flash_attn_paged_args": (V.FlashAttnPagedArgs, ["dst", "lse", "params"]),
              "vtx_kv_score_paged_args": (V.KvScorePagedArgs, ["params", "score_out", "observe", "decay"]),
              "vtx_kv_evict_paged_args": (V.KvEvictPagedArgs, ["next_pos", "kv_len_out", "keep", "out_cap"])}
    body = "".join('printf("%%zu\\n", sizeof(%s));' % n +
                   "".join('printf("%%zu\\n", offsetof(%s, %s));' % (n, f) for f in fs) for n, (_, fs) in probes.items())
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vtx_fa.h"\nint main(void){%s return 0;}\n' % body)
    exe = tmp_path / "p"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    want = []
    for t, fs in probes.values():
        want += [ctypes.sizeof(t)] + [getattr(t, f).offset for f in fs]
    assert got == want


def _kv(kv_type=None, D=128, page=16, Hkv=8, n_pages=10, **kw):
    kv_type = V.F16 if kv_type is None else kv_type
    c = V.VtxPagedKv()
    row = D * 2 if kv_type == V.F16 else D // 32 * 34
    for t, p in ((c.k, 0x10000), (c.v, 0x20000)):
        t.type, t.data = kv_type, p
        for i, (ne, nb) in enumerate(((D, 2 if kv_type == V.F16 else 34), (page, row), (Hkv, page * row), (n_pages, Hkv * page * row))):
            t.ne[i], t.nb[i] = ne, nb
    c.page_table, c.kv_len, c.q_start = 0x1000, 0x2000, 0x3000
    c.n_seq, c.max_pages, c.n_tokens, c.max_new, c.max_kv_len = 2, 4, 2, 1, 4 * page
    for k, v in kw.items():
        if k[:2] in ("k_", "v_"):
            t, f = (c.k if k[0] == "k" else c.v), k[2:]
            if f[:2] in ("ne", "nb") and len(f) == 3:
                getattr(t, f[:2])[int(f[2])] = v
            else:
                setattr(t, f, v)
        else:
            setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(k_type=30), -2), (dict(k_type=V.F32, v_type=V.F32), -2), (dict(v_type=V.Q8_0), -2),
    (dict(D=96), -5), (dict(page=24), -5), (dict(page=8), -5), (dict(page=512), -5),
    (dict(k_data=0), -1), (dict(k_data=0x10008), -4), (dict(k_nb3=8 * 16 * 256 + 8, v_nb3=8 * 16 * 256 + 8), -4),
    (dict(k_nb1=264, v_nb1=264), -4), (dict(v_nb2=16 * 256 + 16), -4), (dict(k_nb1=128, v_nb1=128), -4),
    (dict(kv_type=V.Q8_0, k_nb1=144, v_nb1=144), -4),
    (dict(k_nb3=0, v_nb3=0), -4), (dict(k_nb2=0, v_nb2=0), -4),
    (dict(v_ne3=9), -3), (dict(k_ne2=0, v_ne2=0), -3), (dict(n_seq=-1), -3), (dict(max_kv_len=65), -3),
    (dict(max_new=3), -3), (dict(n_tokens=-1), -3), (dict(max_pages=-1), -3), (dict(kv_len=0), -1), (dict(page_table=0), -1),
]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_cache_refusals_without_device(lib, kw, status):
    c = _kv(**kw)
    a, e = V.KvAppendPagedArgs(), V.KvEvictPagedArgs()
    f, s = V.FlashAttnPagedArgs(), V.KvScorePagedArgs()
    a.freq_base = BASE
    for x in (a, e, f, s):
        x.kv = ctypes.addressof(c)
    assert lib.vtx_kv_append_paged(B(a), None) == status
    assert lib.vtx_flash_attn_paged(B(f), None, 0, None) == status
    assert lib.vtx_kv_score_paged(B(s), None) == status
    assert lib.vtx_kv_evict_paged(B(e), None, 0, None) == status
    none = ctypes.c_size_t(-1).value
    assert lib.vtx_flash_attn_paged_workspace(B(c), 32) == none
    assert lib.vtx_kv_evict_paged_workspace(B(c)) == none


def _tensor(ttype, ne, nb, ptr=0x40000):
    t = V.VtxTensor()
    t.type, t.data = ttype, ptr
    for i in range(4):
        t.ne[i], t.nb[i] = ne[i], nb[i]
    return t


def test_call_refusals_without_device(lib):
    c = _kv()
    keep = [c]

    def params(**kw):
        p = V.params(0.1, causal=True)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def q(**kw):
        t = _tensor(V.F16, [128, 2, 32, 1], [2, 32 * 256, 256, 0])
        for k, v in kw.items():
            if k[:2] in ("ne", "nb") and len(k) == 3:
                getattr(t, k[:2])[int(k[2])] = v
            else:
                setattr(t, k, v)
        return t

    def d(**kw):
        t = _tensor(V.F32, [128, 32, 2, 1], [4, 512, 32 * 512, 0], 0x80000)
        for k, v in kw.items():
            if k[:2] in ("ne", "nb") and len(k) == 3:
                getattr(t, k[:2])[int(k[2])] = v
            else:
                setattr(t, k, v)
        return t

    def attend(qt=None, dt=None, pt=None, ws=0x100000, n=1 << 40, cache=c):
        a = V.FlashAttnPagedArgs()
        ts = [qt or q(), dt or d(), pt or params(), cache]
        keep.append(ts)
        a.kv = ctypes.addressof(cache)
        a.q, a.dst, a.params = (ctypes.addressof(t) for t in ts[:3])
        return lib.vtx_flash_attn_paged(B(a), ws, n, None)

    assert lib.vtx_flash_attn_paged(None, None, 0, None) == -1
    assert attend(q(type=V.Q8_0)) == -2 and attend(q(ne0=64)) == -3 and attend(q(ne1=3)) == -3
    assert attend(q(ne2=20)) == -3                                   # heads do not divide
    assert attend(q(ne2=8 * 17), d(ne1=8 * 17)) == -5                # group above 16
    assert attend(q(nb0=4)) == -4 and attend(q(nb1=8200)) == -4 and attend(q(data=0x40008)) == -4
    assert attend(q(data=0)) == -1 and attend(dt=d(data=0)) == -1
    assert attend(dt=d(type=V.Q8_0)) == -2 and attend(dt=d(ne2=3)) == -3 and attend(dt=d(nb1=516)) == -4
    assert attend(pt=params(max_bias=1.0)) == -5 and attend(pt=params(window=5, causal=0)) == -5
    assert attend(pt=params(scale=float("nan"))) == -5 and attend(pt=params(window=-1)) == -5
    empty = _kv(n_tokens=0, max_new=0)
    assert attend(q(ne1=0), d(ne2=0), cache=empty, ws=0, n=0) in (0, -6)

    def score(**kw):
        a = V.KvScorePagedArgs()
        ts = [q(), params()]
        keep.append(ts)
        a.kv, a.q, a.params = ctypes.addressof(c), ctypes.addressof(ts[0]), ctypes.addressof(ts[1])
        a.lse, a.score, a.score_out, a.row_cap, a.decay = 0x50000, 0x60000, 0x60000, 64, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.vtx_kv_score_paged(B(a), None)

    assert score(row_cap=63) == -3 and score(observe=-1) == -3 and score(lse=0) == -1 and score(score_out=0) == -1
    assert score(score=0) == -1 and score(decay=float("inf")) == -5

    def append(cache=c, **kw):
        a = V.KvAppendPagedArgs()
        a.kv, a.n_head_q, a.q_out_type, a.freq_base, a.row_cap = ctypes.addressof(cache), 32, V.F16, BASE, 64
        a.q, a.q_nb1, a.q_out, a.q_out_nb1 = 0x10000, 32 * 512, 0x20000, 32 * 256
        a.k, a.k_nb1, a.v, a.v_nb1, a.positions, a.row_pos, a.score = 0x30000, 8 * 512, 0x40000, 8 * 512, 0x1000, 0x2000, 0x3000
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.vtx_kv_append_paged(B(a), None)

    assert append(k=0) == -1 and append(positions=0) == -1 and append(q=0) == -1
    assert append(q_out_type=V.Q8_0) == -2 and append(freq_base=0.0) == -5 and append(row_cap=63) == -3
    assert append(k_nb1=8 * 512 - 8) == -4 and append(q=0x10004) == -4 and append(q_out_nb1=32 * 256 - 8) == -4
    assert append(cache=empty) == 0

    def evict(ws=0x100000, n=1 << 40, **kw):
        a = V.KvEvictPagedArgs()
        a.kv, a.score, a.row_pos, a.next_pos, a.kv_len_out = ctypes.addressof(c), 0x10000, 0x20000, 0x30000, 0x40000
        a.keep, a.row_cap, a.out_cap = 32, 64, 32
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.vtx_kv_evict_paged(B(a), ws, n, None)

    assert evict(keep=-1) == -3 and evict(n_sink=20, n_recent=20) == -3 and evict(row_cap=63) == -3
    assert evict(score_out=0x50000, out_cap=31) == -3 and evict(score_out=0x10000) == -3
    assert evict(kv_len_out=0) == -1 and evict(next_pos=0) == -1 and evict(score=0) == -1
    assert evict(ws=0) == -6 and evict(ws=0x100010) == -6 and evict(n=16) == -6


@pytest.mark.parametrize("nb1,nb2", [(0, 0), (512, 0), (256, 32 * 512), (512, 496)])
def test_overlapping_output_rows_are_refused(lib, nb1, nb2):
    c, p = _kv(), V.params(0.1, causal=True)
    q, d = _tensor(V.F16, [128, 2, 32, 1], [2, 32 * 256, 256, 0]), _tensor(V.F32, [128, 32, 2, 1], [4, nb1, nb2, 0], 0x80000)
    a = V.FlashAttnPagedArgs()
    a.kv, a.q, a.dst, a.params = (ctypes.addressof(x) for x in (c, q, d, p))
    assert lib.vtx_flash_attn_paged(B(a), 0x100000, 1 << 40, None) == -4


def test_python_refusals(lib):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    ok = dict(n_tokens=3, max_new=2)
    kv = V.PagedKv(k, k.clone(), i32(2, 2), i32(2), i32(3), 4, **ok)
    with pytest.raises(V.VtxError):
        V.PagedKv(k, k.clone(), i32(2, 2).long(), i32(2), i32(3), 4, **ok)
    with pytest.raises(V.VtxError):
        V.PagedKv(k, k.clone(), i32(2, 2), i32(2), i32(2), 4, **ok)
    with pytest.raises(V.VtxError):
        V.PagedKv(k.float(), k.float(), i32(2, 2), i32(2), i32(3), 4, **ok)
    with pytest.raises(V.VtxError):
        V.PagedKv(k, k.clone(), i32(2, 2), i32(2), i32(3), 3, **ok)          # 3 heads over 2
    with pytest.raises(V.VtxError):
        V.PagedKv(k, k.clone(), i32(2, 2), i32(2), i32(3), 4, n_tokens=3, max_new=2, max_kv_len=33)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(V.VtxError):
        kv.attend(q[:2])
    with pytest.raises(V.VtxError):
        kv.attend(q.double())
    with pytest.raises(V.VtxError):
        kv.attend(q, lse=torch.zeros(4, 3))
    with pytest.raises(V.VtxError):
        kv.score(q, torch.zeros(3, 4), torch.zeros(2, 2, 31))                # fewer entries than rows
    with pytest.raises(V.VtxError):
        kv.evict(torch.zeros(2, 2, 32), 8, row_pos=i32(2, 2, 31))
    with pytest.raises(V.VtxError):
        kv.evict(torch.zeros(2, 2, 32), 8, n_sink=5, n_recent=4)
    with pytest.raises(V.VtxError):
        kv.append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64).half(), i32(3))


def test_reference_forms_agree_with_each_other():
    """The score of rows sums to the visible queries' heads; an eviction keeps a permutation."""
    c = R.build(3, "f16", [(5, 40), (1, 7)], poison=False)
    out, lse, *_ = R.attend(c)
    sc, _ = R.score(c, lse, np.zeros((2, 2, 48)), 48)
    np.testing.assert_allclose(sc[0].sum(), 5 * 8, rtol=1e-9)
    np.testing.assert_allclose(sc[1].sum(), 8, rtol=1e-9)
    src, left = R.evict(c, sc, 10)
    assert left == [10, 7] and all(len(set(v.tolist())) == len(v) for v in src.values())


# ---- on the GPU -------------------------------------------------------------------

def device_kv(c, nhd=False, **kw):
    """(PagedKv, tensors) of a case; nhd: F16 pools with a token's heads adjacent."""
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    pools = [up(c["k_pool"]), up(c["v_pool"])]
    if nhd:
        pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
    new = np.diff(c["start"])
    args = dict(n_tokens=int(c["start"][-1]), max_new=int(new.max()), max_kv_len=int(max(c["len"])))
    args.update(kw)
    kv = V.PagedKv(*pools, up(c["table"]), up(np.array(c["len"], np.int32)), up(c["start"]), c["Hq"], **args)
    return kv


def check_attend(c, got, lse, ref, what=""):
    n_half = 2 if c["kv"] == "q8_0" else 1
    # a Q8_0 cache of 1024 rows or more is unpacked where a stream brings a chunk
    long = c["kv"] == "q8_0" and max(c["len"]) >= 1024 and np.diff(c["start"]).max() * c["Hq"] // c["Hkv"] > 16
    tol, ltol = R.attend_tolerance(ref, n_half, c["D"] if long else 0)
    f16 = got.dtype == torch.float16
    got = got.double().cpu().numpy()
    if f16:
        tol = tol + np.abs(ref[0]) * 2.0 ** -11 + 2.0 ** -25
    bad = ~(np.abs(got - ref[0]) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} out of bounds, first at {np.argwhere(bad)[0]}"
    if lse is not None:
        lse = lse.double().cpu().numpy()
        assert np.array_equal(np.isneginf(lse), np.isneginf(ref[1])), what
        fin = np.isfinite(ref[1])
        off = np.abs(lse[fin] - ref[1][fin])
        assert (off <= ltol[fin]).all(), f"{what}: lse off by {off.max()}"


RAGGED = [(1, 1), (3, 40), (0, 0), (17, 17), (0, 25), (1, 100), (70, 131), (5, 3)]
ATTEND = [
    # kv, streams, Hq, Hkv, D, page, options
    ("f16", [(1, 1)], 8, 2, 128, 16, {}),
    ("f16", [(1, 1023)], 32, 8, 128, 16, {}),
    ("q8_0", [(1, 1023)], 32, 8, 128, 16, {}),
    ("f16", [(1, n) for n in (1, 15, 16, 17, 33, 64, 129, 700, 1500)], 8, 2, 128, 32, {}),
    ("q8_0", [(1, n) for n in (1, 15, 16, 17, 33, 64, 129, 700, 1500)], 8, 2, 128, 32, {}),
    ("f16", [(4, 300), (2, 2), (1, 31), (4, 1000)], 8, 2, 128, 16, {}),
    ("q8_0", [(4, 300), (2, 2), (1, 31), (4, 1000)], 8, 2, 64, 16, {}),
    ("f16", RAGGED, 8, 2, 128, 16, {}),
    ("q8_0", RAGGED, 8, 2, 128, 64, {}),
    ("f16", RAGGED, 4, 4, 64, 32, {}),
    ("f16", RAGGED, 15, 5, 64, 128, {}),
    ("q8_0", RAGGED, 15, 5, 128, 16, {}),
    ("f16", RAGGED, 16, 1, 128, 256, {}),
    ("q8_0", [(1, 90), (3, 70)], 16, 1, 64, 16, {}),
    ("f16", RAGGED, 8, 2, 128, 16, dict(window=20)),
    ("q8_0", RAGGED, 8, 2, 128, 16, dict(window=1)),
    ("f16", [(1, 900), (2, 400), (300, 700)], 8, 2, 128, 16, dict(window=130)),
    ("f16", RAGGED, 8, 2, 128, 16, dict(softcap=5.0)),
    ("q8_0", RAGGED, 8, 2, 64, 16, dict(softcap=3.0, window=33)),
    ("f16", RAGGED, 8, 2, 128, 16, dict(causal=False)),
    ("f16", [(391, 391)], 32, 8, 128, 64, {}),
    ("f16", [(300, 1300), (129, 129), (1, 2000)], 8, 2, 128, 64, {}),
    ("q8_0", [(200, 900), (129, 129)], 8, 2, 128, 32, {}),
    ("f16", [(64, 1999)], 4, 4, 64, 16, {}),
    ("q8_0", [(90, 1500), (1, 700), (0, 30), (40, 40), (1, 3)], 8, 2, 128, 16, {}),
    ("q8_0", [(90, 1500), (33, 1025)], 5, 5, 64, 32, dict(window=300)),
    ("q8_0", [(300, 1200)], 15, 5, 128, 128, dict(softcap=10.0)),
    ("f16", [(33, 3000)], 8, 1, 64, 128, {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_attend(i):
    kv_type, streams, Hq, Hkv, D, page, opt = ATTEND[i]
    c = R.build(100 + i, kv_type, streams, Hq, Hkv, D, page)
    ref = R.attend(c, **opt)
    kw = {("logit_softcap" if k == "softcap" else k): v for k, v in opt.items()}
    q = torch.from_numpy(c["q"]).cuda()
    for nhd in ((False, True) if kv_type == "f16" else (False,)):
        kv = device_kv(c, nhd)
        for dt in (torch.float32, torch.float16):
            out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
            lse = torch.full(q.shape[:2], 7.0, device="cuda")
            kv.attend(q, out=out, lse=lse, **kw)
            check_attend(c, out, lse, ref, f"{ATTEND[i]} nhd={nhd} {dt}")
    assert V.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type,streams", [("f16", [(1, 50), (2, 9)]), ("f16", [(90, 150), (1, 33)]), ("q8_0", [(40, 90)])])
def test_attend_strided_and_f32_q(kv_type, streams):
    """F32 q (rounded to half by the kernel), token and head strides, rows outside the batch left alone."""
    c = R.build(7, kv_type, streams)
    T, Hq, D = c["q"].shape
    ref = R.attend(c)
    kv = device_kv(c)
    q = torch.from_numpy(c["q"]).cuda()
    wide = torch.randn(T, Hq, 2, D, device="cuda")
    wide[:, :, 1] = q.float()
    big = torch.full((T + 2, Hq + 1, D), 3.0, device="cuda")
    kv.attend(wide[:, :, 1], out=big[1:T + 1, :Hq])
    check_attend(c, big[1:T + 1, :Hq], None, ref)
    assert (big[0] == 3).all() and (big[T + 1] == 3).all() and (big[:, Hq] == 3).all()
    h = torch.empty(Hq, T, D, dtype=torch.float16, device="cuda")         # head-major
    kv.attend(q.transpose(0, 1).contiguous().transpose(0, 1), out=h.transpose(0, 1))
    check_attend(c, h.transpose(0, 1), None, ref)


@pytest.mark.gpu
def test_attend_tokens_of_no_stream_and_default_bounds():
    """Tokens behind the last stream are left alone; bounds may be loose."""
    c = R.build(8, "f16", [(2, 40), (30, 64)])
    ref = R.attend(c)
    kv = device_kv(c, n_tokens=40, max_new=40, max_kv_len=None)
    q = torch.full((40, 8, 128), float("nan"), dtype=torch.float16, device="cuda")
    q[:32] = torch.from_numpy(c["q"])
    out = torch.full((40, 8, 128), 5.0, device="cuda")
    kv.attend(q, out=out)
    check_attend(c, out[:32], None, ref)
    assert (out[32:] == 5).all() and V.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
def test_attend_longer_than_its_bound(kv_type):
    """A kv_len above max_kv_len is still attended to in full."""
    c = R.build(9, kv_type, [(1, 900), (1, 20), (20, 700)])
    kv = device_kv(c, max_kv_len=64)
    out = kv.attend(torch.from_numpy(c["q"]).cuda())
    check_attend(c, out, None, R.attend(c))


@pytest.mark.gpu
def test_more_new_tokens_than_the_bound_are_reported():
    c = R.build(10, "f16", [(40, 60), (1, 30)])
    kv = device_kv(c, max_new=1)
    out = torch.zeros(41, 8, 128, device="cuda")
    kv.attend(torch.from_numpy(c["q"]).cuda(), out=out)
    assert V.read_device_error() == 41
    ref = R.attend(c)
    assert np.abs(out[40].cpu().numpy() - ref[0][40]).max() < 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("streams", [[(1, 60)], [(40, 60)]])
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
def test_bad_pages_are_reported(kv_type, streams):
    """A table entry outside the pool, and a length beyond the table: an error word, no access outside."""
    c = R.build(11, kv_type, streams, poison=False)
    q = torch.from_numpy(c["q"]).cuda()
    for bad in (-1, 1 << 30, c["k_pool"].shape[0]):
        kv = device_kv(c)
        kv.page_table[0, 1] = bad
        lse = torch.empty(q.shape[:2], device="cuda")
        kv.attend(q, lse=lse)
        assert V.read_device_error() == 40
        kv.score(q, lse, torch.zeros(1, 2, 64, device="cuda"))
        assert V.read_device_error() == 40
        before = kv.k_pool.clone()
        n = q.shape[0]
        kv.append(torch.randn(n, 2, 128, device="cuda"), torch.randn(n, 2, 128, device="cuda"),
                  torch.arange(n, dtype=torch.int32, device="cuda"))
        err = V.read_device_error()
        assert err == (40 if 60 - n < 32 else 0)
        changed = (kv.k_pool != before).any(3).any(1)
        rows = {(int(kv.page_table[0, r // 16]), r % 16) for r in range(60 - n, 60) if r // 16 != 1}
        assert {tuple(x) for x in changed.nonzero().tolist()} <= rows
    kv = device_kv(c)
    kv.kv_len.fill_(1 << 20)
    kv.page_table.fill_(0)
    kv.attend(q)
    assert V.read_device_error() == 41


@pytest.mark.gpu
def test_attend_far_pages():
    """Page offsets beyond 32 bits."""
    n_pages = 34000                                    # x 4 x 256 x 64 halves: 4.5e9 bytes a pool
    c = R.build(12, "f16", [(1, 300), (40, 500)], 8, 4, 64, 256, poison=False)
    k = torch.zeros(n_pages, 4, 256, 64, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    m = c["k_pool"].shape[0]
    k[-m:], v[-m:] = torch.from_numpy(c["k_pool"]).cuda(), torch.from_numpy(c["v_pool"]).cuda()
    assert k.stride(0) * 2 * (n_pages - m) > 2 ** 32
    table = torch.from_numpy(c["table"] + (n_pages - m)).int().cuda()
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = V.PagedKv(k, v, table, up(c["len"]), up(c["start"]), 8, n_tokens=41, max_new=40, max_kv_len=500)
    check_attend(c, kv.attend(torch.from_numpy(c["q"]).cuda()), None, R.attend(c))


APPEND = [("f16", 128, 16, [(1, 1), (1, 100), (0, 7), (5, 40), (3, 2)], 8, 2), ("q8_0", 128, 32, [(1, 33), (40, 64), (2, 2)], 8, 2),
          ("q8_0", 64, 16, [(1, 5), (7, 30)], 5, 5), ("f16", 64, 256, [(600, 700)], 2, 1), ("f16", 128, 64, [(1, i + 1) for i in range(300)], 32, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(APPEND)))
@pytest.mark.parametrize("qdt", [torch.float16, torch.float32])
def test_append(i, qdt):
    kv_type, D, page, streams, Hq, Hkv = APPEND[i]
    c = R.build(200 + i, kv_type, streams, Hq, Hkv, D, page, poison=False)
    rng = np.random.default_rng(i)
    T = c["q"].shape[0]
    q, k, v = (rng.standard_normal((T, h, D)).astype(np.float32) for h in (Hq, Hkv, Hkv))
    pos = rng.integers(0, 200000, T).astype(np.int32)
    kv = device_kv(c)
    up = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    cap = max(c["len"]) + 3
    sc, rp = torch.full((len(streams), Hkv, cap), 9.0, device="cuda"), torch.full((len(streams), Hkv, cap), -9, dtype=torch.int32, device="cuda")
    q_out = torch.empty(T, Hq, D, dtype=qdt, device="cuda")
    kv.append(up(k), up(v), up(pos), BASE, q=up(q), q_out=q_out, row_pos=rp, score=sc)
    yq, yk = R.rope(q, pos, BASE), R.rope(k, pos, BASE)
    mag = lambda x: np.abs(x.reshape(*x.shape[:-1], -1, 2)).sum(-1).repeat(2, -1)  # noqa: E731
    # an angle and a rotation in f32: (|x0| + |x1|) * 2^-21; then one rounding to the stored type
    eps = np.abs(yq) * (2.0 ** -11 if qdt == torch.float16 else 2.0 ** -24) + 2.0 ** -25
    assert (np.abs(q_out.double().cpu().numpy() - yq) <= mag(q) * 2.0 ** -21 + eps).all()
    want_k, want_v = c["k_pool"].copy(), c["v_pool"].copy()
    got_k, got_v = kv.k_pool.cpu().numpy(), kv.v_pool.cpu().numpy()
    want_sc, want_rp = np.full(sc.shape, 9.0), np.full(rp.shape, -9)
    for s, n in enumerate(c["len"]):
        t0, t1 = c["start"][s], c["start"][s + 1]
        for t in range(t0, t1):
            r = n - (t1 - t)
            if r < 0:
                continue
            p, w = c["table"][s, r // page], r % page
            want_sc[s, :, r], want_rp[s, :, r] = 0.0, pos[t]
            for got, y, x in ((got_k[p, :, w], yk[t], mag(k[t])), (got_v[p, :, w], v[t].astype(np.float64), 0 * v[t])):
                if kv_type == "f16":
                    assert (np.abs(got.astype(np.float64) - y) <= x * 2.0 ** -21 + np.abs(y) * 2.0 ** -11 + 2.0 ** -25).all()
                else:       # half a step of the block's scale, which is itself a half
                    amax = np.abs(y.reshape(Hkv, -1, 32)).max(-1, keepdims=True).repeat(32, -1).reshape(y.shape)
                    assert (np.abs(R.q8_to_f64(got) - y) <= amax / 127 * 0.501 + amax * 2.0 ** -11 + x * 2.0 ** -21).all()
            got_k[p, :, w], got_v[p, :, w] = want_k[p, :, w], want_v[p, :, w]
    assert np.array_equal(got_k.view(np.uint8), want_k.view(np.uint8)) and np.array_equal(got_v.view(np.uint8), want_v.view(np.uint8))
    assert np.array_equal(sc.cpu().numpy(), want_sc) and np.array_equal(rp.cpu().numpy(), want_rp)
    assert V.read_device_error() == 0


SCORE = [("f16", [(1, 1)], 8, 2, 128, 16, {}), ("f16", RAGGED, 8, 2, 128, 16, {}), ("q8_0", RAGGED, 8, 2, 128, 64, {}),
         ("f16", RAGGED, 15, 5, 64, 32, dict(window=20)), ("q8_0", RAGGED, 16, 1, 64, 16, dict(softcap=5.0)),
         ("f16", RAGGED, 8, 2, 128, 16, dict(causal=False)), ("f16", [(100, 600), (1, 40)], 8, 2, 128, 16, dict(observe=32)),
         ("f16", [(1, 2000), (1, 300)], 32, 8, 128, 16, dict(decay=0.5)), ("q8_0", [(1, 700)], 32, 8, 128, 16, {}),
         ("f16", [(300, 1500)], 8, 2, 128, 64, dict(decay=0.0)), ("q8_0", [(300, 1500), (2, 90)], 8, 2, 128, 64, {}),
         ("q8_0", [(200, 400)], 15, 5, 64, 16, dict(window=50)), ("f16", [(60, 5000)], 32, 16, 64, 128, {}), ("f16", [(70, 300)], 4, 4, 64, 16, dict(window=100, observe=9))]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(SCORE)))
def test_score(i):
    kv_type, streams, Hq, Hkv, D, page, opt = SCORE[i]
    c = R.build(300 + i, kv_type, streams, Hq, Hkv, D, page)
    att = {k: v for k, v in opt.items() if k in ("window", "softcap", "causal")}
    lse = R.attend(c, **att)[1].astype(np.float32)
    cap = max(c["len"]) + 5
    old = np.random.default_rng(i).random((len(streams), Hkv, cap)).astype(np.float32)
    want, tol = R.score(c, lse, old, cap, **opt)
    kw = {("logit_softcap" if k == "softcap" else k): v for k, v in opt.items()}
    kv = device_kv(c)
    q, ls = torch.from_numpy(c["q"]).cuda(), torch.from_numpy(lse).cuda()
    a = torch.from_numpy(old).cuda()
    b = torch.full_like(a, -4.0)
    kv.score(q, ls, a, score_out=b, **kw)
    kv.score(q, ls, a, **kw)
    live = np.arange(cap)[None, None] < np.array(c["len"])[:, None, None]
    live = np.broadcast_to(live, old.shape)
    for got, rest in ((a, old), (b, np.full_like(old, -4.0))):
        got = got.cpu().numpy()
        assert np.array_equal(got[~live], rest[~live])
        bad = live & ~(np.abs(got - want) <= tol)
        assert not bad.any(), f"{SCORE[i]}: {bad.sum()} of {live.sum()}, worst {np.abs(got - want)[live].max()}"
    assert V.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
@pytest.mark.parametrize("streams", [[(2, 50), (1, 9)], [(80, 500), (1, 33)]])
def test_score_f32_strided_q(kv_type, streams):
    c = R.build(14, kv_type, streams)
    lse = R.attend(c)[1].astype(np.float32)
    want, tol = R.score(c, lse, np.zeros((2, 2, 512)), 512)
    kv = device_kv(c)
    T, Hq, D = c["q"].shape
    wide = torch.randn(T, Hq, 2, D, device="cuda")
    wide[:, :, 1] = torch.from_numpy(c["q"]).cuda().float()
    for q in (wide[:, :, 1], wide.half()[:, :, 1]):
        got = torch.zeros(2, 2, 512, device="cuda")
        kv.score(q, torch.from_numpy(lse).cuda(), got)
        assert (np.abs(got.cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
def test_append_rows_aligned_to_eight_bytes():
    """Token strides and bases of 8 bytes: the same bits as 16-byte aligned rows."""
    for kv_type, D in (("f16", 128), ("q8_0", 128), ("f16", 64), ("q8_0", 64)):
        c = R.build(15, kv_type, [(3, 40), (1, 7)], 8, 2, D, poison=False)
        rng = np.random.default_rng(2)
        x = {h: torch.from_numpy(rng.standard_normal((4, h * D)).astype(np.float32)).cuda() for h in (8, 2)}
        pos = torch.tensor([5, 6, 7, 900], dtype=torch.int32, device="cuda")
        got = []
        for pad in (0, 2):
            kv = device_kv(c)
            wide = {h: torch.zeros(4, v.shape[1] + 2 * pad, device="cuda") for h, v in x.items()}
            view = {}
            for h, v in x.items():
                wide[h][:, pad:pad + v.shape[1]] = v
                view[h] = wide[h][:, pad:pad + v.shape[1]].unflatten(1, (h, D))
            out = torch.zeros(4, 8 * D + 2 * pad, device="cuda")[:, pad:pad + 8 * D].unflatten(1, (8, D))
            half = torch.zeros(4, 8 * D + 4 * pad, dtype=torch.float16, device="cuda")[:, 2 * pad:2 * pad + 8 * D].unflatten(1, (8, D))
            kv.append(view[2], view[2], pos, q=view[8], q_out=out)
            kv.append(view[2], view[2], pos, q=view[8], q_out=half)
            got.append((kv.k_pool.clone(), kv.v_pool.clone(), out.clone(), half.clone()))
        for a, b in zip(*got):
            assert torch.equal(a, b)
    # rotated in place
    kv = device_kv(c)
    q = view[8].clone()
    kv.append(view[2], view[2], pos, q=q, q_out=q)
    assert torch.equal(q, got[0][2])


@pytest.mark.gpu
@pytest.mark.parametrize("streams,D,kw,opt", [
    ([(30, 90), (1, 60), (17, 17)], 128, {}, {}),                            # short: the pages as they are
    ([(95, 95)], 64, {}, dict(softcap=4.0)),
    ([(33, 96), (1, 900), (129, 1401)], 128, {}, {}),                        # unpacked
    ([(200, 777), (5, 5), (0, 40)], 64, {}, dict(window=100)),
    ([(70, 640)], 128, {}, dict(softcap=4.0)),
    ([(70, 640)], 64, {}, dict(causal=False)),
    ([(140, 700), (1, 300)], 128, dict(max_kv_len=1 << 21), {}),             # too large a copy for the bound
    ([(140, 700), (1, 300)], 64, dict(max_kv_len=1 << 22), {}),
])
def test_attend_q8_chunks_round_p_alone(streams, D, kw, opt):
    """Chunks over Q8_0 caches: neither K nor V is rounded, only P (in the short
    form P times 64 times V's scale, whose subnormals cost up to 2^-25 / 64 of a
    scale, 2 |v| for scales of 1/64 and more)."""
    c = R.build(31, "q8_0", streams, 8, 2, D, 16)
    if kw:                                                  # as many pages as the bound asks for
        wide = np.zeros((len(streams), kw["max_kv_len"] // 16), np.int32)
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
    q = torch.from_numpy(c["q"]).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    kv = device_kv(c, **kw)
    ref = R.attend(c, **opt)
    tol, ltol = R.attend_tolerance(ref, 1)
    named = {("logit_softcap" if k == "softcap" else k): v for k, v in opt.items()}
    out = kv.attend(q, lse=lse, out=torch.empty_like(q, dtype=torch.float32), **named).double().cpu().numpy()
    assert (np.abs(out - ref[0]) <= tol + ref[4] * 2.0 ** -24).all()
    fin = np.isfinite(ref[1])
    assert (np.abs(lse.cpu().numpy()[fin] - ref[1][fin]) <= ltol[fin]).all()
    assert V.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
@pytest.mark.parametrize("new,D,Hq,Hkv,opt", [
    (20, 128, 8, 2, {}), (33, 64, 8, 2, dict(window=190)), (17, 128, 8, 8, dict(causal=False)),
    (9, 64, 16, 1, dict(softcap=4.0)), (40, 128, 8, 2, {})])
def test_attend_one_query_tile(kv_type, new, D, Hq, Hkv, opt):
    """One Q tile over an odd and an even number of key tiles, alone and together, one
    stream with fewer rows than tokens."""
    lengths = [new, 127, 128, 200, 300, 500, 650, 1300, 7]
    c = R.build(37, kv_type, [(new, n) for n in lengths], Hq, Hkv, D, 32)
    q, named = torch.from_numpy(c["q"]).cuda(), {("logit_softcap" if k == "softcap" else k): v for k, v in opt.items()}
    ref = R.attend(c, **opt)
    tol, ltol = R.attend_tolerance(ref, 1)
    # Q8_0 below 96 rows: P is rounded after V's scale went in, with subnormals of its own
    tol = tol + ref[4] * 2.0 ** -24
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda")
    lse = torch.empty(q.shape[:2], device="cuda")
    one, one_lse = torch.empty_like(out), torch.empty_like(lse)
    kv = device_kv(c)
    kv.attend(q, out=out, lse=lse, **named)
    for s, n in enumerate(lengths):
        rows = slice(s * new, (s + 1) * new)
        alone = V.PagedKv(kv.k_pool, kv.v_pool, up(c["table"][s:s + 1]), up(np.array([n], np.int32)),
                          up(np.array([0, new], np.int32)), Hq, n_tokens=new, max_new=new, max_kv_len=n)
        alone.attend(q[rows].float(), out=one[rows], lse=one_lse[rows], **named)
    for o, e in ((out, lse), (one, one_lse)):
        o, e = o.double().cpu().numpy(), e.double().cpu().numpy()
        assert (np.abs(o - ref[0]) <= tol).all()
        fin = np.isfinite(ref[1])
        assert np.array_equal(np.isneginf(e), ~fin) and (np.abs(e[fin] - ref[1][fin]) <= ltol[fin]).all()
    assert V.read_device_error() == 0


@pytest.mark.gpu
def test_unpacked_cache_past_its_bound():
    """A chunk over a Q8_0 cache that is unpacked: lengths up to whole pages above
    max_kv_len are served, longer ones reported."""
    c = R.build(16, "q8_0", [(40, 1100)])
    q = torch.from_numpy(c["q"]).cuda()
    check_attend(c, device_kv(c, max_kv_len=1030).attend(q), None, R.attend(c))
    assert V.read_device_error() == 0
    c = R.build(17, "q8_0", [(40, 1500)])
    device_kv(c, max_kv_len=1030).attend(q)
    assert V.read_device_error() == 41


@pytest.mark.gpu
def test_many_streams_and_none():
    """More streams than a search step holds, most without tokens; and no stream at all."""
    rng = np.random.default_rng(0)
    streams = [(int(n), int(n + k)) for n, k in zip(rng.choice([0, 0, 0, 1, 2, 9], 150), rng.integers(0, 60, 150))]
    c = R.build(18, "f16", streams, 4, 1, 64)
    kv = device_kv(c)
    q = torch.from_numpy(c["q"]).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    ref = R.attend(c)
    check_attend(c, kv.attend(q, lse=lse), lse, ref)
    T = q.shape[0]
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    rows = torch.zeros(150, 1, max(c["len"]), dtype=torch.int32, device="cuda") - 1
    kv.append(torch.randn(T, 1, 64, device="cuda"), torch.randn(T, 1, 64, device="cuda"), pos, row_pos=rows)
    want = np.full(rows.shape, -1)
    for s, n in enumerate(c["len"]):
        new = c["start"][s + 1] - c["start"][s]
        want[s, 0, n - new:n] = np.arange(c["start"][s], c["start"][s + 1])
    assert np.array_equal(rows.cpu().numpy(), want) and V.read_device_error() == 0
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    none = V.PagedKv(kv.k_pool, kv.v_pool, i32(0, 1), i32(0), i32(1), 4, n_tokens=0, max_new=0)
    assert none.attend(q[:0]).shape == (0, 4, 64)
    none.append(torch.zeros(0, 1, 64, device="cuda"), torch.zeros(0, 1, 64, device="cuda"), i32(0))
    none.score(q[:0], lse[:0], torch.zeros(0, 1, 16, device="cuda"))
    none.evict(torch.zeros(0, 1, 16, device="cuda"), 8)


@pytest.mark.gpu
def test_score_of_streams_without_tokens_only_decays():
    c = R.build(19, "f16", [(0, 30), (0, 0), (0, 17)])
    kv = device_kv(c, n_tokens=0, max_new=0)
    a = torch.rand(3, 2, 32, device="cuda")
    b = kv.score(torch.zeros(0, 8, 128, dtype=torch.float16, device="cuda"), torch.zeros(0, 8, device="cuda"), a,
                 score_out=torch.full_like(a, -1.0), decay=0.5)
    for s, n in enumerate(c["len"]):
        assert torch.equal(b[s, :, :n], a[s, :, :n] * 0.5) and (b[s, :, n:] == -1).all()


@pytest.mark.gpu
def test_calls_on_streams_of_their_own():
    """Two caches worked on from two streams at once, repeatedly: each as alone."""
    cases = [R.build(20, "f16", [(1, 1500), (1, 700), (30, 600)], 8, 2), R.build(21, "q8_0", [(1, 1800), (1, 40)], 8, 2)]
    kvs, qs = [device_kv(c) for c in cases], [torch.from_numpy(c["q"]).cuda() for c in cases]
    alone = [kv.attend(q) for kv, q in zip(kvs, qs)]
    side = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[torch.empty_like(a) for _ in range(20)] for a in alone]
    for i in range(20):
        for kv, q, s, o in zip(kvs, qs, side, outs):
            kv.attend(q, out=o[i], stream=s)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert all(torch.equal(a, x) for x in o)


def run_evict(c, sc, keep, in_place=False, row_pos=None, next_pos=None, **kw):
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    kv = device_kv(c, max_new=0, n_tokens=0)
    cap = sc.shape[2]
    t = {"score": up(sc), "pos": up(row_pos) if row_pos is not None else None}
    nxt = up(np.asarray(next_pos, np.int32)) if next_pos is not None else None
    if in_place:
        so, po = t["score"], t["pos"]
        src = torch.full(sc.shape, -7, dtype=torch.int32, device="cuda")
        n = kv.evict(t["score"], keep, row_pos=t["pos"], next_pos=nxt, score_out=so, pos_out=po, src_out=src, **kw)
    else:
        out_cap = max(keep, 1) + 2
        so = torch.full((*sc.shape[:2], out_cap), -7.0, device="cuda")
        po = torch.full((*sc.shape[:2], out_cap), -7, dtype=torch.int32, device="cuda")
        src = torch.full_like(po, -7)
        n = torch.empty(len(c["len"]), dtype=torch.int32, device="cuda")
        kv.evict(t["score"], keep, n, row_pos=t["pos"], next_pos=nxt, score_out=so, pos_out=po, src_out=src, **kw)
    src_ref, left = R.evict(c, sc, keep, row_pos=row_pos, next_pos=next_pos, **kw)
    assert n.tolist() == left
    page = c["page"]
    k, v = c["k_pool"].copy(), c["v_pool"].copy()
    for (s, h), new in src_ref.items():
        m = len(new)
        assert np.array_equal(src[s, h, :m].cpu().numpy(), new)
        assert np.array_equal(so[s, h, :m].cpu().numpy(), sc[s, h, new], equal_nan=True)
        if po is not None:
            assert np.array_equal(po[s, h, :m].cpu().numpy(), new if row_pos is None else row_pos[s, h, new])
        if not in_place:
            assert (so[s, h, m:] == -7).all() and (po[s, h, m:] == -7).all() and (src[s, h, m:] == -7).all()
        old_k, old_v = (R.rows_of(c[p], c["table"][s], c["len"][s])[h] for p in ("k_pool", "v_pool"))
        for r in range(m):
            p = c["table"][s, r // page]
            k[p, h, r % page], v[p, h, r % page] = old_k[new[r]], old_v[new[r]]
    assert np.array_equal(kv.k_pool.cpu().numpy().view(np.uint8), k.view(np.uint8))
    assert np.array_equal(kv.v_pool.cpu().numpy().view(np.uint8), v.view(np.uint8))
    assert V.read_device_error() == 0
    return kv


EVICT = [("f16", [100, 30, 0, 1, 64, 65], 64, 128, 16), ("q8_0", [100, 30, 0, 1, 64, 65], 64, 128, 16),
         ("q8_0", [333, 2], 100, 64, 32), ("f16", [2500], 700, 64, 128), ("f16", [50, 20], 0, 64, 16),
         ("f16", [300], 1, 128, 16), ("f16", [1025, 1024, 1023], 1023, 128, 64), ("f16", [9000], 4000, 64, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(EVICT)))
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(i, kind):
    kv_type, lens, keep, D, page = EVICT[i]
    c = R.build(400 + i, kv_type, [(0, n) for n in lens], 4, 2, D, page, poison=False)
    rng = np.random.default_rng(i)
    cap = max(lens) + 1
    sc = rng.standard_normal((len(lens), 2, cap)).astype(np.float32)
    if kind == "ties":
        sc = np.round(sc)
    if kind == "odd":
        sc = rng.choice(np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-45, -3.4e38, 1.0], np.float32), sc.shape)
    pos = np.sort(rng.choice(4 * cap, (cap,), replace=False))[None, None].repeat(len(lens), 0).repeat(2, 1).astype(np.int32)
    pos = rng.permuted(pos, axis=2) if kind == "random" else pos
    nxt = [int(pos[s, 0, :n].max()) + 1 if n else 0 for s, n in enumerate(lens)]
    run_evict(c, sc, keep)
    run_evict(c, sc, keep, n_sink=min(4, keep), n_recent=min(20, max(keep - 4, 0)))
    run_evict(c, sc, keep, row_pos=pos, next_pos=nxt, n_sink=min(40, keep // 2), n_recent=keep // 3)
    run_evict(c, sc, keep, in_place=True, row_pos=pos, next_pos=nxt, n_sink=min(3, keep))


@pytest.mark.gpu
def test_evict_more_rows_than_fit_in_shared_memory():
    n = 48 * 1024 + 77
    c = {"D": 64, "Hq": 1, "Hkv": 1, "page": 256, "kv": "f16", "len": [n], "start": np.zeros(2, np.int32),
         "table": np.random.default_rng(0).permutation(-(-n // 256)).astype(np.int32)[None]}
    rng = np.random.default_rng(1)
    c["k_pool"] = rng.standard_normal((-(-n // 256), 1, 256, 64)).astype(np.float16)
    c["v_pool"] = rng.standard_normal(c["k_pool"].shape).astype(np.float16)
    run_evict(c, np.round(rng.standard_normal((1, 1, n)) * 20).astype(np.float32), 20000, n_sink=4, n_recent=100)


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused():
    """Every tensor of a call is checked to lie where the pools do, before any launch."""
    c = R.build(33, "f16", [(2, 20)])
    kv = device_kv(c)
    q, pos = torch.from_numpy(c["q"]).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    k, sc = torch.zeros(2, 2, 128, device="cuda"), torch.zeros(1, 2, 32, device="cuda")
    lse, n = torch.zeros(2, 8, device="cuda"), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: V.PagedKv(kv.k_pool, kv.v_pool.cpu(), kv.page_table, kv.kv_len, kv.q_start, 8, n_tokens=2, max_new=2),
                 lambda: V.PagedKv(kv.k_pool, kv.v_pool, kv.page_table, kv.kv_len.cpu(), kv.q_start, 8, n_tokens=2, max_new=2),
                 lambda: kv.append(k.cpu(), k, pos), lambda: kv.append(k, k.cpu(), pos), lambda: kv.append(k, k, pos.cpu()),
                 lambda: kv.append(k, k, pos, q=q.float().cpu()), lambda: kv.append(k, k, pos, q=q.float(), q_out=q.cpu()),
                 lambda: kv.append(k, k, pos, score=sc.cpu()), lambda: kv.append(k, k, pos, row_pos=sc.int().cpu()),
                 lambda: kv.attend(q.cpu()), lambda: kv.attend(q, out=q.cpu()), lambda: kv.attend(q, lse=lse.cpu()),
                 lambda: kv.score(q, lse.cpu(), sc), lambda: kv.score(q, lse, sc.cpu()),
                 lambda: kv.score(q, lse, sc, score_out=sc.cpu()), lambda: kv.evict(sc.cpu(), 8),
                 lambda: kv.evict(sc, 8, n), lambda: kv.evict(sc, 8, next_pos=n), lambda: kv.evict(sc, 8, src_out=sc.int().cpu())):
        with pytest.raises(V.VtxError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("streams", [[(6, 4), (2, 30)], [(40, 30), (1, 9)]])
def test_widest_window_is_none(streams):
    """The largest window, with streams of more tokens than rows too."""
    c = R.build(34, "f16", streams)
    q = torch.from_numpy(c["q"]).cuda()
    T = q.shape[0]
    outs = []
    for w in (0, 2 ** 31 - 1):
        kv, lse = device_kv(c), torch.empty(T, 8, device="cuda")
        out = kv.attend(q, lse=lse, window=w)
        sc = [kv.score(x, lse, torch.zeros(2, 2, 64, device="cuda"), window=w) for x in (q, q.float())]
        outs.append([out, lse, *sc])
    ref = R.attend(c)
    check_attend(c, outs[1][0], outs[1][1], ref)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
def test_append_rotates_queries_of_no_stream():
    """q_out is written for every token, with K and V going nowhere."""
    c = R.build(35, "f16", [(3, 20)])
    kv = device_kv(c)
    q, k, pos = torch.randn(3, 8, 128).cuda(), torch.randn(3, 2, 128).cuda(), torch.tensor([5, 6, 900], dtype=torch.int32).cuda()
    want = kv.append(k, k, pos, q=q)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    none = V.PagedKv(kv.k_pool, kv.v_pool, i32(0, 1), i32(0), i32(1), 8, n_tokens=3, max_new=0)
    before = kv.k_pool.clone()
    assert torch.equal(none.append(k, k, pos, q=q), want)
    kv.q_start.zero_()
    assert torch.equal(kv.append(k, k, pos, q=q), want)
    assert torch.equal(kv.k_pool.view(torch.int16), before.view(torch.int16)) and V.read_device_error() == 0


@pytest.mark.gpu
def test_evict_lengths_over_next_pos():
    """kv_len_out may be next_pos: every head still protects the recent rows."""
    rng = np.random.default_rng(36)
    c = R.build(36, "f16", [(0, 900)] * 40, 8, 4, 64)
    sc = torch.from_numpy(rng.random((40, 4, 900), np.float32)).cuda()
    got = []
    for alias in (False, True):
        kv = device_kv(c, n_tokens=0, max_new=0)
        nxt = kv.kv_len.clone()
        src = torch.zeros(40, 4, 100, dtype=torch.int32, device="cuda")
        n = kv.evict(sc, 100, nxt if alias else kv.kv_len.clone(), n_recent=64, next_pos=nxt, src_out=src)
        got.append((n.cpu(), src.cpu()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and (got[0][0] == 100).all()


@pytest.mark.gpu
def test_evict_reports_a_length_above_its_bound():
    c = R.build(13, "f16", [(0, 100), (0, 40)], 4, 2, 64, poison=False)
    kv = device_kv(c, max_kv_len=64, n_tokens=0, max_new=0)
    before = kv.k_pool.clone()
    n = kv.evict(torch.rand(2, 2, 64, device="cuda"), 40, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert V.read_device_error() == 41 and n.tolist() == [100, 40]
    assert torch.equal(kv.k_pool, before)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
def test_run_of_all_four_in_a_graph(kv_type):
    """Prompt, then decode steps replayed from one captured graph, an eviction
    whenever the budget is passed: every step's attention and scores against
    the 64-bit forms on the cache as it then is."""
    Hq, Hkv, D, page, cap, n = 8, 2, 128, 16, 96, 2
    rng = np.random.default_rng(5)
    W = D * 2 if kv_type == "f16" else D // 32 * 34
    pools = [torch.zeros(14, Hkv, page, W, dtype=torch.uint8, device="cuda") for _ in range(2)]
    if kv_type == "f16":
        pools = [p.view(torch.float16) for p in pools]
    table = torch.from_numpy(rng.permutation(14)[:12].reshape(2, 6).astype(np.int32)).cuda()
    kv_len = torch.zeros(n, dtype=torch.int32, device="cuda")
    score = torch.zeros(n, Hkv, cap, device="cuda")
    row_pos = torch.zeros(n, Hkv, cap, dtype=torch.int32, device="cuda")

    def host(q, new):
        return {"D": D, "Hq": Hq, "Hkv": Hkv, "page": page, "kv": kv_type, "len": kv_len.tolist(),
                "table": table.cpu().numpy(), "start": np.concatenate([[0], np.cumsum(new)]).astype(np.int32),
                "k_pool": pools[0].cpu().numpy(), "v_pool": pools[1].cpu().numpy(), "q": q.cpu().numpy()}

    new = [70, 33]
    start = torch.tensor([0, 70, 103], dtype=torch.int32, device="cuda")
    prompt = V.PagedKv(*pools, table, kv_len, start, Hq, n_tokens=103, max_new=70)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    kv_len += torch.tensor(new, dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(x, dtype=torch.int32, device="cuda") for x in new])
    q = prompt.append(f(103, Hkv, D), f(103, Hkv, D), pos, BASE, q=f(103, Hq, D), row_pos=row_pos, score=score)
    lse = torch.empty(103, Hq, device="cuda")
    c = host(q, new)
    check_attend(c, prompt.attend(q, lse=lse), lse, R.attend(c))
    old = score.cpu().numpy()
    prompt.score(q, lse, score, observe=16)
    want, tol = R.score(c, lse.cpu().numpy(), old, cap, observe=16)
    assert (np.abs(score.cpu().numpy() - want) <= tol).all()

    step = V.PagedKv(*pools, table, kv_len, torch.arange(n + 1, dtype=torch.int32, device="cuda"), Hq, n_tokens=n, max_new=1)
    k, v, qf = (torch.empty(n, h, D, device="cuda") for h in (Hkv, Hkv, Hq))
    q16, out, lse = torch.empty(n, Hq, D, dtype=torch.float16, device="cuda"), torch.empty(n, Hq, D, device="cuda"), torch.empty(n, Hq, device="cuda")
    positions = torch.tensor(new, dtype=torch.int32, device="cuda")

    def one():
        kv_len.add_(1)
        step.append(k, v, positions, BASE, q=qf, q_out=q16, row_pos=row_pos, score=score)
        step.attend(q16, out=out, lse=lse)
        step.score(q16, lse, score, decay=0.9)
        positions.add_(1)

    side = torch.cuda.Stream()
    graph = None
    for t in range(30):
        for x in (k, v, qf):
            x.copy_(f(*x.shape))
        before = score.clone()
        if graph is None:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            state = [x.clone() for x in (kv_len, positions, score)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                one()
            for x, y in zip((kv_len, positions, score), state):
                assert torch.equal(x, y)                      # capturing ran nothing
        else:
            graph.replay()
        c = host(q16, [1, 1])
        check_attend(c, out, lse, R.attend(c), f"step {t}")
        old = before.cpu().numpy()
        for s, m in enumerate(c["len"]):
            old[s, :, m - 1] = 0.0
        want, tol = R.score(c, lse.cpu().numpy(), old, cap, decay=0.9)
        assert (np.abs(score.cpu().numpy() - want) <= tol).all(), f"step {t}"
        if max(c["len"]) > 80:
            src, left = R.evict(c, score.cpu().numpy(), 60, 4, 10, row_pos.cpu().numpy(), positions.tolist())
            rows = {key: R.rows_of(c["k_pool"], c["table"][key[0]], c["len"][key[0]])[key[1]][m] for key, m in src.items()}
            step.evict(score, 60, n_sink=4, n_recent=10, row_pos=row_pos, next_pos=positions, score_out=score, pos_out=row_pos)
            assert kv_len.tolist() == left
            after = pools[0].cpu().numpy()
            for (s, h), want_rows in rows.items():
                assert np.array_equal(R.rows_of(after, c["table"][s], left[s])[h], want_rows)
    assert V.read_device_error() == 0
