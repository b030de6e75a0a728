"""The paged decoder cache at the edges of what its header allows."""
import threading
import time

import numpy as np
import pytest

import paged_ref as R
import vtx_attn as V
from test_paged import ATTEND, BASE, device_kv

torch = pytest.importorskip("torch")


def up(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# Q8_0: P carries V's scale d when it is rounded, so a subnormal loses 2^-25 of a product
# whose largest is 16 d or more; with the cases' scales of 1/127 and more that is 2^-22 of
# what a whole weight would give
SUBNORMAL = 2.0 ** -22


def close(got, want, tol):
    got = got.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - want) <= tol) | (np.isneginf(got) & np.isneginf(want)))
    assert not bad.any(), f"{bad.sum()} of {bad.size} out of bounds, first at {np.argwhere(bad)[0]}"


# ---- a kv_len above the table's capacity --------------------------------------------

def beyond(seed, kv_type, streams, page, *shape):
    """A case whose tables end at their last whole page, and its lengths with `streams`' third entries added."""
    c = R.build(seed, kv_type, [x[:2] for x in streams], *shape, page, poison=False)
    most = max(c["len"]) // page
    c["table"] = np.ascontiguousarray(c["table"][:, :most])
    c["len"] = [x[1] + x[2] for x in streams]
    return c, most * page


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
@pytest.mark.parametrize("new,over", [(1, 1), (1, 40), (3, 1), (5, 3), (40, 7), (40, 90)])
def test_append_beyond_the_table_is_dropped(kv_type, new, over):
    """Token i of n goes to row kv_len - n + i; one at or behind the capacity is
    dropped and reported, and the rows in front of it are not touched."""
    c, cap = beyond(50, kv_type, [(new, 64, over), (2, 30, 0)], 16, 8, 2, 128)
    kv = device_kv(c, max_kv_len=cap)
    before = [p.clone() for p in (kv.k_pool, kv.v_pool)]
    f = lambda h: torch.randn(new + 2, h, 128, device="cuda")  # noqa: E731
    score, row_pos = torch.full((2, 2, cap), 9.0, device="cuda"), torch.full((2, 2, cap), -9, dtype=torch.int32, device="cuda")
    k, v, pos = f(2), f(2), torch.arange(1000, 1002 + new, dtype=torch.int32, device="cuda")
    kv.append(k, v, pos, BASE, row_pos=row_pos, score=score)
    assert V.read_device_error() == 41
    want_pos = np.full((2, 2, cap), -9)
    for t in range(new):
        if cap + over - new + t < cap:
            want_pos[0, :, cap + over - new + t] = 1000 + t
    want_pos[1, :, 28:30] = [1000 + new, 1001 + new]
    assert np.array_equal(row_pos.cpu().numpy(), want_pos)
    assert np.array_equal(score.cpu().numpy(), np.where(want_pos >= 0, 0.0, 9.0))
    written = {(int(c["table"][s, r // 16]), r % 16) for s in (0, 1) for r in np.flatnonzero(want_pos[s, 0] >= 0)}
    for now, old in zip((kv.k_pool, kv.v_pool), before):
        changed = (now.view(torch.uint8) != old.view(torch.uint8)).any(3).any(1)
        assert {tuple(x) for x in changed.nonzero().tolist()} == written


BEYOND = [
    ("f16", [(1, 64, 3), (2, 30, 0)], 8, 2, 128, {}), ("q8_0", [(4, 64, 2), (1, 64, 9)], 8, 2, 64, {}),
    ("f16", [(1, 960, 5)], 8, 2, 128, dict(window=40)), ("f16", [(4, 64, 40), (1, 20, 0)], 8, 2, 128, dict(window=20)),
    ("f16", [(40, 64, 9), (1, 33, 0)], 8, 2, 128, {}), ("f16", [(300, 960, 100)], 8, 2, 64, dict(window=130)),
    ("f16", [(40, 64, 60)], 8, 2, 128, dict(window=10)), ("f16", [(40, 64, 9), (3, 50, 0)], 8, 2, 128, dict(causal=False)),
    ("q8_0", [(40, 64, 9), (1, 33, 0)], 8, 2, 128, {}), ("q8_0", [(40, 64, 60)], 8, 2, 128, dict(window=10)),
    ("q8_0", [(90, 960, 20), (1, 100, 0)], 8, 2, 64, {}), ("q8_0", [(90, 960, 70)], 8, 2, 128, dict(window=50)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(BEYOND)))
def test_attend_and_score_beyond_the_table(i):
    """A stream longer than its table keeps its tokens' rows: each sees the rows that exist of those it may see."""
    kv_type, streams, Hq, Hkv, D, opt = BEYOND[i]
    c, cap = beyond(60 + i, kv_type, streams, 16, Hq, Hkv, D)
    kv = device_kv(c, max_kv_len=cap)
    q = up(c["q"])
    lse = torch.empty(q.shape[:2], device="cuda")
    out = kv.attend(q, lse=lse, **opt)
    assert V.read_device_error() == 41
    ref = R.attend(c, **opt)
    tol, ltol = R.attend_tolerance(ref, 1)
    close(out, ref[0], tol + ref[4] * SUBNORMAL)
    close(lse, ref[1], ltol)
    c["len"] = [min(n, cap) for n in c["len"]]                # rows that the sums run over
    for x in (q, q.float()):
        got = kv.score(x, up(ref[1].astype(np.float32)), torch.zeros(len(streams), Hkv, cap, device="cuda"), **opt)
        assert V.read_device_error() == 41
        want, stol = score_beyond(c, streams, ref[1].astype(np.float32), cap, opt)
        close(got, want, stol)


def score_beyond(c, streams, lse, cap, opt):
    """R.score with the rows' offsets of the uncut lengths."""
    want, tol = np.zeros((2, len(streams), c["Hkv"], cap))
    for s, (new, n, over) in enumerate(streams):
        one = dict(c, len=[n + over], table=c["table"][s:s + 1], start=np.array([0, new], np.int32),
                   q=c["q"][c["start"][s]:c["start"][s + 1]])
        wide = cap + over                                       # entries behind the table stay 0
        kr = R.values(R.rows_of(c["k_pool"], c["table"][s], c["len"][s]))
        rows = c["len"][s]
        for h in range(c["Hq"]):
            q = one["q"][:, h].astype(np.float64)
            k = kr[h // (c["Hq"] // c["Hkv"])]
            x = R.scores(q, k, n + over - new, c["D"] ** -0.5, opt.get("causal", True), opt.get("window", 0), 0.0)
            ls = lse[c["start"][s]:c["start"][s + 1], h].astype(np.float64)[:, None]
            with np.errstate(invalid="ignore"):
                p = np.where(np.isneginf(ls) | np.isneginf(x), 0.0, np.exp(x - ls))
            e = (c["D"] + 8) * 2.0 ** -24 * c["D"] ** -0.5 * (np.abs(q) @ np.abs(k).T)
            e = e + 2.0 ** -20 * (1 + np.where(np.isinf(x), 0, np.abs(x)) + np.abs(np.where(np.isinf(ls), 0, ls)))
            g = h // (c["Hq"] // c["Hkv"])
            want[s, g, :rows] += p.sum(0)
            tol[s, g, :rows] += (p * e).sum(0)
        assert wide >= rows
    return want, tol + np.abs(want) * 2.0 ** -20 + 1e-30


# ---- scores that are not finite ---------------------------------------------------------

# streaming: one split and many, drafts; chunks: one Q tile, pairs, splits; short and unpacked Q8_0
FINITE = [("f16", [(1, 60), (3, 50)], 8, 2, 128), ("f16", [(1, 3000)], 8, 2, 64), ("q8_0", [(2, 700), (1, 9)], 8, 2, 128),
          ("f16", [(40, 300), (1, 70)], 8, 2, 64), ("f16", [(40, 300)], 8, 2, 128), ("f16", [(33, 2500)], 8, 2, 64),
          ("f16", [(33, 2500)], 8, 2, 128), ("f16", [(700, 700)], 20, 20, 64), ("f16", [(700, 700)], 20, 20, 128),
          ("q8_0", [(40, 80)], 8, 2, 64), ("q8_0", [(40, 300), (20, 120)], 8, 2, 64), ("q8_0", [(33, 2500)], 8, 2, 128)]


def finite_case(i):
    kv_type, streams, Hq, Hkv, D = FINITE[i]
    c = R.build(80 + i, kv_type, streams, Hq, Hkv, D, 16)
    ref = R.attend(c)
    tol, ltol = R.attend_tolerance(ref, 1)
    return c, ref, tol + ref[4] * SUBNORMAL, ltol


def check_finite(c, kv, q, ref, tol, ltol, nan, what):
    """Rows of `nan` (tokens, heads) hold NaN throughout, the others what the reference says."""
    out, lse = torch.full(q.shape, 3.0, device="cuda"), torch.full(q.shape[:2], 3.0, device="cuda")
    kv.attend(q, out=out, lse=lse)
    o, e = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.array_equal(np.isnan(e), nan), f"{what}: lse NaN at {np.argwhere(np.isnan(e) != nan)[:4]}"
    assert np.isnan(o[nan]).all(), f"{what}: {(~np.isnan(o[nan])).sum()} values of NaN rows are not NaN"
    close(out[up(~nan)], ref[0][~nan], tol[~nan])
    close(lse[up(~nan)], ref[1][~nan], ltol[~nan])
    return lse


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(FINITE)))
def test_query_rows_of_nan(i):
    """A NaN in a query row: its result and lse are NaN, as are the scores of the rows it sees; no other changes."""
    c, ref, tol, ltol = finite_case(i)
    kv, q = device_kv(c), up(c["q"])
    T, Hq, D = q.shape
    G = Hq // c["Hkv"]
    for t, h, d in ((0, 1, slice(None)), (T - 1, Hq - 1, 5), (T // 2, 0, D - 1)):
        bad = q.clone()
        bad[t, h, d] = float("nan")
        nan = np.zeros((T, Hq), bool)
        nan[t, h] = True
        lse = check_finite(c, kv, bad, ref, tol, ltol, nan, f"{FINITE[i]} token {t}")
        s = int(np.searchsorted(c["start"][1:], t, side="right"))
        sc = kv.score(bad, lse, torch.zeros(len(c["len"]), c["Hkv"], max(c["len"]), device="cuda"))
        want = np.zeros(sc.shape, bool)
        want[s, h // G, :c["len"][s] - (c["start"][s + 1] - t) + 1] = True
        assert np.array_equal(torch.isnan(sc).cpu().numpy(), want)
    assert V.read_device_error() == 0


def set_key(kv, c, s, row, value):
    """Sets a key's first value (F16) or first scale (Q8_0); returns what undoes it."""
    page, at = int(c["table"][s, row // c["page"]]), row % c["page"]
    old = kv.k_pool[page, :, at].clone()
    if c["kv"] == "f16":
        kv.k_pool[page, :, at, 0] = value
    else:
        kv.k_pool[page, :, at, :2] = torch.tensor([value], dtype=torch.float16).view(torch.uint8).cuda()

    def undo():
        kv.k_pool[page, :, at] = old
    return undo


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(FINITE)))
def test_keys_of_nan(i):
    """A NaN key makes NaN of every token that sees it, wherever in a tile it stands, and of no other."""
    c, ref, tol, ltol = finite_case(i)
    kv, q = device_kv(c), up(c["q"])
    for s, n in enumerate(c["len"]):
        new = int(c["start"][s + 1] - c["start"][s])
        for row in sorted({0, 6, 7, 14, n // 3, n // 2 | 7, n - new, n - 1} & set(range(n))):
            undo = set_key(kv, c, s, row, float("nan"))
            nan = np.zeros(q.shape[:2], bool)
            nan[c["start"][s]:c["start"][s + 1]] = (row <= n - new + np.arange(new))[:, None]
            check_finite(c, kv, q, ref, tol, ltol, nan, f"{FINITE[i]} stream {s} row {row}")
            undo()
    assert V.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("i", [i for i, x in enumerate(FINITE) if x[0] == "f16"])
def test_infinite_scores(i):
    """A score of +inf makes NaN of its token's result and lse, one of -inf counts nothing."""
    c, _, _, _ = finite_case(i)
    c["q"][:, :, 0] = np.where(np.random.default_rng(i).random(c["q"].shape[:2]) < 0.3, 1, -1)
    _, _, _, err, _ = R.attend(c)
    kv, q = device_kv(c), up(c["q"])
    s, n = len(c["len"]) - 1, c["len"][-1]
    new = int(c["start"][s + 1] - c["start"][s])
    for row in sorted({0, 7, n // 2 | 6, n - 1} & set(range(n))):
        far = dict(c, k_pool=c["k_pool"].copy())               # a weight of exactly 0 where q is -1
        far["k_pool"][c["table"][s, row // 16], :, row % 16, 0] = 60000
        out, lse, a, _, tiny = R.attend(far)
        alone = c["start"][s] + row - (n - new) if row == 0 else -1      # the token that sees this key and no other
        if alone >= c["start"][s]:
            down = c["q"][alone, :, 0] < 0
            out[alone, down], lse[alone, down] = 0.0, -np.inf
        ref = (out, lse, a, err, tiny)
        tol, ltol = R.attend_tolerance(ref, 1)
        undo = set_key(kv, c, s, row, float("inf"))
        nan = np.zeros(q.shape[:2], bool)
        t = slice(c["start"][s], c["start"][s + 1])
        nan[t] = (row <= n - new + np.arange(new))[:, None] & (c["q"][t, :, 0] > 0)
        check_finite(c, kv, q, ref, tol + ref[4] * SUBNORMAL, ltol, nan, f"{FINITE[i]} row {row}")
        undo()
    assert V.read_device_error() == 0


# ---- one workspace under several descriptors ------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
def test_one_workspace_for_prompts_and_steps(kv_type):
    """Descriptors of other bounds, sizes and streams take turns on one workspace
    that was zeroed once: a split chunk, a split step of one token, many
    streams, a chunk beside tokens; twice."""
    cases = [R.build(90, kv_type, x, 8, 2) for x in ([(40, 2000)], [(1, 2000)], [(1, 900 + 50 * i) for i in range(9)],
                                                     [(30, 700), (1, 1500), (2, 600)], [(3, 2500)])]
    kvs = [device_kv(c) for c in cases]
    ws = torch.zeros(max(kv.workspace.numel() for kv in kvs), dtype=torch.uint8, device="cuda")
    for kv in kvs:
        kv._ws = (ws.data_ptr(), ws.numel())
    refs = [R.attend(c) for c in cases]
    for _ in range(2):
        for c, kv, ref in zip(cases, kvs, refs):
            q = up(c["q"])
            out, lse = torch.full(q.shape, 7.0, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
            kv.attend(q, out=out, lse=lse)
            tol, ltol = R.attend_tolerance(ref, 1)
            close(out, ref[0], tol + ref[4] * SUBNORMAL)
            close(lse, ref[1], ltol)
    assert V.read_device_error() == 0


@pytest.mark.gpu
def test_results_repeat_themselves():
    """The same call gives the same bits, whatever ran in between."""
    for kv_type in ("f16", "q8_0"):
        for streams in ([(1, 1500)] * 5, [(200, 1500), (1, 900), (3, 40)], [(391, 391)], [(20, 3000)]):
            c = R.build(95, kv_type, streams, 8, 2)
            kv, q = device_kv(c), up(c["q"])
            first = kv.attend(q)
            for _ in range(5):
                assert torch.equal(first, kv.attend(q))


# ---- results made on another stream -----------------------------------------------------------

class FakeStreams:
    """torch.cuda's streams and allocations on a machine without a GPU: which
    stream was current when a tensor was made, and which others were noted on it."""

    def __init__(self, monkeypatch):
        self.current, self.made, self.noted = ["main"], [], []
        empty, here = torch.empty, self

        class Context:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(self):
                here.current.append(self.stream)

            def __exit__(self, *_):
                here.current.pop()

        def fake_empty(*shape, **kw):
            kw["device"] = "cpu"
            here.made.append(here.current[-1])
            return empty(*shape, **kw)

        monkeypatch.setattr(torch.cuda, "stream", Context)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: here.current[-1])
        monkeypatch.setattr(torch, "empty", fake_empty)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: here.noted.append(s), raising=False)


class SideStream:
    cuda_stream = 77


def host_kv(call, n_seq=1, n_tokens=2):
    """A PagedKv over host memory whose calls go to `call(args, ...)`."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    kv = V.PagedKv(k, k.clone(), i32(n_seq, 2), i32(n_seq), i32(n_seq + 1), 4, n_tokens=n_tokens, max_new=n_tokens)

    class Lib:
        vtx_flash_attn_paged = vtx_kv_append_paged = vtx_kv_score_paged = vtx_kv_evict_paged = staticmethod(call)

    kv._lib, kv.dev, kv._only = Lib, torch.device("cuda"), True
    return kv


def test_results_come_from_the_memory_of_the_stream_that_writes_them(monkeypatch):
    """A block of the current stream's memory may still be in use there; a result
    for another stream is made in that stream's, and the current one noted on it."""
    kv = host_kv(lambda *_: 0)
    q, k, pos = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    side = SideStream()
    fake = FakeStreams(monkeypatch)
    kv.attend(q, stream=side)
    kv.append(k, k, pos, q=q, stream=side)
    assert fake.made == [side, side] and fake.noted == ["main", "main"] and fake.current == ["main"]


@pytest.mark.gpu
def test_results_made_for_another_stream_are_their_own():
    """Work queued on the current stream writes a block that was freed a moment ago;
    a call on another stream with a result of that size is not touched by it."""
    c = R.build(96, "f16", [(20, 300), (1, 700)], 8, 2)
    kv, q = device_kv(c), up(c["q"])
    T = q.shape[0]
    k, pos, qf = torch.randn(T, 2, 128, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda"), q.float()
    want, want_q = kv.attend(q), kv.append(k, k, pos, q=qf)
    want = kv.attend(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)
        for like in (want, want_q):
            busy = torch.empty_like(like)
            busy.fill_(7)
            del busy
        out, got_q = kv.attend(q, stream=side), kv.append(k, k, pos, q=qf, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got_q, want_q)


# ---- calls from several host threads ------------------------------------------------------------

def test_calls_of_two_host_threads_do_not_mix():
    """Every call reaches the library with its own arguments, before and after a while inside it."""
    seen = []

    def tensors(a):
        if isinstance(a, V.KvAppendPagedArgs):
            return a.k, a.q_out or 0
        if isinstance(a, V.KvEvictPagedArgs):
            return a.score, a.keep
        q = V.VtxTensor.from_address(a.q).data
        return (q, V.VtxTensor.from_address(a.dst).data) if isinstance(a, V.FlashAttnPagedArgs) else (q, a.score)

    def call(args, *_):
        before = tensors(args._obj)
        time.sleep(0.003)
        seen.append((before, tensors(args._obj)))
        return 0

    kv = host_kv(call)
    pos, stream = torch.zeros(2, dtype=torch.int32), SideStream()
    want, fails = [], []

    def work(n):
        q, out, lse, k, score = torch.zeros(2, 4, 64), torch.zeros(2, 4, 64), torch.zeros(2, 4), torch.zeros(2, 2, 64), torch.zeros(1, 2, 32)
        keep.append((q, out, lse, k, score))
        try:
            for _ in range(5):
                kv.attend(q, out=out, stream=stream)
                if n == 0:
                    kv.append(k, k, pos, stream=stream)
                else:
                    kv.append(k, k, pos, q=q, q_out=out, stream=stream)
                kv.score(q, lse, score, stream=stream)
                kv.evict(score, n + 3, stream=stream)
        except Exception as e:  # noqa: BLE001
            fails.append(e)
        want.extend(5 * [(q.data_ptr(), out.data_ptr()), (k.data_ptr(), out.data_ptr() if n else 0),
                         (q.data_ptr(), score.data_ptr()), (score.data_ptr(), n + 3)])

    keep = []
    threads = [threading.Thread(target=work, args=(n,)) for n in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails and all(a == b for a, b in seen)
    assert sorted(a for a, _ in seen) == sorted(want)


# ---- axes of one element --------------------------------------------------------------------------

def one_token(h, dtype=torch.float32, device="cpu", kind=0):
    """A (1, h, 64) view of one token whose first stride is not a token's."""
    x = torch.randn(h, 64, device=device, dtype=dtype)
    if kind == 0:
        return x.unsqueeze(1).transpose(0, 1)              # head-major: strides (64, 64, 1)
    return x.unsqueeze(2).permute(2, 0, 1)                 # strides (1, 64, 1)


@pytest.mark.parametrize("kind", [0, 1])
def test_strides_of_one_token_are_its_own(kind):
    """The stride of an axis with one element means nothing and is not passed on."""
    got = []

    def call(args, *_):
        a = args._obj
        if isinstance(a, V.KvAppendPagedArgs):
            got.append((a.k_nb1, a.v_nb1, a.q_nb1, a.q_out_nb1))
        else:
            q, d = (V.VtxTensor.from_address(x) for x in (a.q, a.dst))
            got.append((q.nb[1], q.nb[2], d.nb[2], d.nb[1]))
        return 0

    kv, side = host_kv(call, n_tokens=1), SideStream()
    q, k, pos = one_token(4, kind=kind), one_token(2, kind=kind), torch.zeros(1, dtype=torch.int32)
    kv.append(k, k, pos, q=q, q_out=one_token(4, torch.float16, kind=kind), stream=side)
    kv.attend(q, out=one_token(4, torch.float16, kind=kind), stream=side)
    assert got == [(512, 512, 1024, 512), (1024, 256, 512, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
def test_one_token_of_any_stride(kind):
    c = R.build(97, "f16", [(1, 40)], 4, 1, 64)
    kv, kv2 = device_kv(c), device_kv(c)
    q, k, pos = one_token(4, device="cuda", kind=kind), one_token(1, device="cuda", kind=kind), torch.full((1,), 9, dtype=torch.int32, device="cuda")
    q16 = kv.append(k, k, pos, q=q)
    want = kv.attend(q16)
    out, half = one_token(4, device="cuda", kind=kind), one_token(4, torch.float16, "cuda", kind)
    plain = lambda x: x.clone(memory_format=torch.contiguous_format)  # noqa: E731
    kv2.append(plain(k), plain(k), pos, q=plain(q), q_out=half)
    kv2.attend(half, out=out)
    assert torch.equal(half, q16) and torch.equal(out, want)
    assert torch.equal(kv.k_pool.view(torch.int16), kv2.k_pool.view(torch.int16))


# ---- chunks next to single tokens, replayed -----------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
def test_mixed_steps_replayed_with_other_lengths(kv_type):
    """A captured step whose single tokens run beside its chunks: every replay
    goes by the lengths, pages and queries written just before it."""
    rng = np.random.default_rng(3)
    streams = [(40, 600), (1, 900), (2, 500), (20, 300), (1, 40)]
    c = R.build(98, kv_type, streams, 8, 2, poison=False)
    kv = device_kv(c)
    q = up(c["q"])
    out, lse = torch.empty(q.shape, device="cuda"), torch.empty(q.shape[:2], device="cuda")
    new_len, new_table, new_q = kv.kv_len.clone(), kv.page_table.clone(), q.clone()

    def step():
        kv.kv_len.copy_(new_len)
        kv.page_table.copy_(new_table)
        q.copy_(new_q)
        kv.attend(q, out=out, lse=lse)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    pages = c["k_pool"].shape[0]
    for _ in range(8):
        c["len"] = [int(rng.integers(n, most + 1)) for n, most in streams]
        c["table"] = rng.integers(0, pages, c["table"].shape).astype(np.int32)
        c["q"] = rng.standard_normal(c["q"].shape).astype(np.float16)
        new_len.copy_(torch.tensor(c["len"], dtype=torch.int32))
        new_table.copy_(up(c["table"]))
        new_q.copy_(up(c["q"]))
        graph.replay()
        ref = R.attend(c)
        tol, ltol = R.attend_tolerance(ref, 1)
        close(out, ref[0], tol + ref[4] * SUBNORMAL)
        close(lse, ref[1], ltol)
    assert V.read_device_error() == 0


# ---- layers that share their lengths ---------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 1500])
def test_layers_with_one_kv_len_evict_by_the_old_lengths(n):
    """Each layer's eviction reads the shared lengths and writes the new ones
    elsewhere; every layer keeps its own best rows."""
    cases = [R.build(110 + i, "f16", [(0, n), (0, 40), (0, n - 90)], 4, 2, 64, 16, poison=False) for i in range(3)]
    kvs = [device_kv(c, n_tokens=0, max_new=0) for c in cases]
    kv_len, left = kvs[0].kv_len.clone(), torch.zeros(3, dtype=torch.int32, device="cuda")
    kvs = [V.PagedKv(kv.k_pool, kv.v_pool, kv.page_table, kv_len, kv.q_start, 4, n_tokens=0, max_new=0, max_kv_len=n) for kv in kvs]
    rng = np.random.default_rng(4)
    scores = [rng.random((3, 2, n)).astype(np.float32) for _ in cases]
    srcs = [torch.full((3, 2, 100), -1, dtype=torch.int32, device="cuda") for _ in cases]
    for kv, sc, src in zip(kvs, scores, srcs):
        kv.evict(up(sc), 100, left, n_sink=4, n_recent=20, src_out=src)
    kv_len.copy_(left)
    assert kv_len.tolist() == [100, 40, 100]
    for c, kv, sc, src in zip(cases, kvs, scores, srcs):
        want, _ = R.evict(c, sc, 100, 4, 20)
        pools = [(c[p], getattr(kv, p).cpu().numpy()) for p in ("k_pool", "v_pool")]
        for (s, h), rows in want.items():
            assert np.array_equal(src[s, h, :len(rows)].cpu().numpy(), rows)
            for old, now in pools:
                kept = R.rows_of(now, c["table"][s], len(rows))[h]
                assert np.array_equal(kept, R.rows_of(old, c["table"][s], c["len"][s])[h][rows])
    assert V.read_device_error() == 0


# ---- shared workspaces ---------------------------------------------------------------------------------

def test_share_takes_the_workspaces_of_another():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)

    def make(n_seq, max_pages, **kw):
        return V.PagedKv(k, k.clone(), i32(n_seq, max_pages), i32(n_seq), i32(n_seq + 1), 4, n_tokens=40, max_new=40, **kw)

    big = make(8, 64)
    small = make(1, 20, share=big)
    assert small.workspace is big.workspace and small._ws == big._ws and small._evict_ws == big._evict_ws
    assert make(8, 64, share=small).workspace is big.workspace
    own = make(1, 20)
    assert own.workspace is not big.workspace and own.workspace.numel() < big.workspace.numel()
    with pytest.raises(V.VtxError) as e:
        make(8, 64, share=own)
    assert e.value.status == -6
    with pytest.raises(V.VtxError) as e:                  # more counters than their fixed place holds
        make(1, 1, share=make(40000, 2))
    assert e.value.status == -6


@pytest.mark.gpu
def test_layers_and_steps_share_one_set():
    """A prompt and then single tokens through three layers over one set of workspaces."""
    cases = [R.build(120 + i, "q8_0", [(60, 700), (33, 600)], 8, 2, poison=False) for i in range(3)]
    first, layers = None, []
    for c in cases:
        kv = device_kv(c, share=first)
        first = first or kv
        one = dict(c, start=np.array([0, 1, 2], np.int32), q=c["q"][:2])
        layers.append((c, kv, one, V.PagedKv(kv.k_pool, kv.v_pool, kv.page_table, kv.kv_len, up(one["start"]), 8,
                                             n_tokens=2, max_new=1, max_kv_len=700, share=first)))
    for _ in range(2):
        for what in (0, 2):
            for l in layers:
                c, kv = l[what], l[what + 1]
                out = kv.attend(up(c["q"]))
                ref = R.attend(c)
                close(out, ref[0], R.attend_tolerance(ref, 1)[0] + ref[4] * SUBNORMAL)
    for i, (c, kv, _, _) in enumerate(layers):
        sc = np.random.default_rng(i).random((2, 2, 700)).astype(np.float32)
        src = torch.empty(2, 2, 200, dtype=torch.int32, device="cuda")
        kv.evict(up(sc), 200, torch.zeros(2, dtype=torch.int32, device="cuda"), src_out=src)
        for (s, h), rows in R.evict(c, sc, 200)[0].items():
            assert np.array_equal(src[s, h].cpu().numpy(), rows)
    assert V.read_device_error() == 0


# ---- Q8_0 caches: P is all that is rounded ----------------------------------------------------------------

Q8_CASES = [i for i, x in enumerate(ATTEND) if x[0] == "q8_0"]


def q8_tolerance(c, ref):
    """Bounds with one rounding to half, P's, which carries V's scale d: relative 2^-11, and
    2^-25 for a subnormal, of a product whose largest is 16 d or more in the streaming
    kernel, 64 d over short caches, 1 over an unpacked one (whose V is exact to 2^-25)."""
    tol, ltol = R.attend_tolerance(ref, 1)
    scales = R.half_bits_to_f64(c["v_pool"].reshape(*c["v_pool"].shape[:-1], -1, R.QB)[..., :2])
    low = np.abs(scales[np.isfinite(scales)]).min()
    return tol + ref[4] * 2.0 ** -25 / min(1.0, 16 * low) + 2.0 ** -25, ltol


def test_q8_bounds_notice_a_rounded_key():
    """K rounded to half would move a score by 2^-12 of its products' sum: more than lse's bound."""
    c = R.build(100 + Q8_CASES[1], "q8_0", [(1, 1), (1, 15), (1, 64)], 8, 2, 128, 32)
    ref = R.attend(c)
    _, ltol = q8_tolerance(c, ref)
    out = np.zeros(ref[1].shape)
    for s, n in enumerate(c["len"]):
        k = R.values(R.rows_of(c["k_pool"], c["table"][s], n)).astype(np.float16).astype(np.float64)
        for h in range(8):
            x = k[h // 4] @ c["q"][s, h].astype(np.float64) * 128 ** -0.5
            out[s, h] = np.log(np.exp(x - x.max()).sum()) + x.max()
    assert (np.abs(out - ref[1]) > ltol).mean() > 0.25


@pytest.mark.gpu
@pytest.mark.parametrize("i", Q8_CASES)
def test_attend_over_q8_rounds_p_alone(i):
    kv_type, streams, Hq, Hkv, D, page, opt = ATTEND[i]
    c = R.build(100 + i, kv_type, streams, Hq, Hkv, D, page)
    ref = R.attend(c, **opt)
    tol, ltol = q8_tolerance(c, ref)
    q = up(c["q"])
    out, lse = torch.empty(q.shape, device="cuda"), torch.empty(q.shape[:2], device="cuda")
    device_kv(c).attend(q, out=out, lse=lse, **{("logit_softcap" if k == "softcap" else k): v for k, v in opt.items()})
    close(out, ref[0], tol)
    close(lse, ref[1], ltol)


# ---- all four calls in one captured step ---------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "q8_0"])
@pytest.mark.parametrize("in_place", [False, True])
def test_captured_step_with_its_eviction(kv_type, in_place):
    """A step of append, attention, score and eviction captured once and replayed:
    single tokens next to a chunk, each stream brought back to its budget."""
    Hq, Hkv, D, page, cap, keep = 8, 2, 128, 16, 128, 70
    rng = np.random.default_rng(6)
    new, length = [1, 30, 1], [60, 50, 69]
    c = R.build(130, kv_type, [(n, cap) for n in new], Hq, Hkv, D, page, poison=False)
    c["table"], c["len"], T = np.ascontiguousarray(c["table"][:, :cap // page]), length, sum(new)
    kv = device_kv(c, max_kv_len=cap)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    k, v, qf = (torch.zeros(T, h, D, device="cuda") for h in (Hkv, Hkv, Hq))
    q16, out, lse = torch.zeros(T, Hq, D, dtype=torch.float16, device="cuda"), torch.zeros(T, Hq, D, device="cuda"), torch.zeros(T, Hq, device="cuda")
    score, row_pos = torch.zeros(3, Hkv, cap, device="cuda"), torch.arange(cap, dtype=torch.int32, device="cuda").repeat(3, Hkv, 1)
    score += f(3, Hkv, cap).abs()
    n_new, positions = torch.tensor(new, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    next_pos, left = torch.tensor(length, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    src = torch.zeros(3, Hkv, cap, dtype=torch.int32, device="cuda")
    within = torch.cat([torch.arange(n, dtype=torch.int32) for n in new]).cuda()
    which = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).cuda()
    state = {}

    def step():
        positions.copy_(next_pos[which] + within)
        kv.kv_len.add_(n_new)
        next_pos.add_(n_new)
        kv.append(k, v, positions, BASE, q=qf, q_out=q16, row_pos=row_pos, score=score)
        kv.attend(q16, out=out, lse=lse)
        kv.score(q16, lse, score, observe=8)
        for name, x in (("k_pool", kv.k_pool), ("v_pool", kv.v_pool), ("score", score), ("pos", row_pos), ("len", kv.kv_len)):
            state.setdefault(name, torch.zeros_like(x)).copy_(x)          # before the eviction
        kv.evict(score, keep, None if in_place else left, n_sink=4, n_recent=40, row_pos=row_pos, next_pos=next_pos,
                 score_out=score, pos_out=row_pos, src_out=src)
        if not in_place:
            kv.kv_len.copy_(left)

    graph = None
    for turn in range(8):
        for x in (k, v, qf):
            x.copy_(f(*x.shape))
        if graph is None:
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        else:
            old = score.clone()
            graph.replay()
        host = {n: x.cpu().numpy() for n, x in state.items()}
        now = dict(c, len=host["len"].tolist(), q=q16.cpu().numpy(), k_pool=host["k_pool"], v_pool=host["v_pool"])
        ref = R.attend(now)
        tol, ltol = R.attend_tolerance(ref, 1)
        close(out, ref[0], tol + ref[4] * SUBNORMAL)
        close(lse, ref[1], ltol)
        if turn:
            before = old.cpu().numpy()
            for s, n in enumerate(now["len"]):
                before[s, :, n - new[s]:n] = 0.0
            want, stol = R.score(now, lse.cpu().numpy(), before, cap, observe=8)
            for s, n in enumerate(now["len"]):
                assert (np.abs(host["score"][s, :, :n] - want[s, :, :n]) <= stol[s, :, :n]).all()
        rows, lens = R.evict(now, host["score"], keep, 4, 40, host["pos"], next_pos.tolist())
        assert kv.kv_len.tolist() == lens
        after = [(host[p], getattr(kv, p).cpu().numpy()) for p in ("k_pool", "v_pool")]
        for (s, h), r in rows.items():
            assert np.array_equal(src[s, h, :len(r)].cpu().numpy(), r)
            assert np.array_equal(score[s, h, :len(r)].cpu().numpy(), host["score"][s, h, r])
            assert np.array_equal(row_pos[s, h, :len(r)].cpu().numpy(), host["pos"][s, h, r])
            for was, is_ in after:
                assert np.array_equal(R.rows_of(is_, c["table"][s], len(r))[h],
                                      R.rows_of(was, c["table"][s], now["len"][s])[h][r])
    assert V.read_device_error() == 0
