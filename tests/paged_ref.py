"""Plain 64-bit forms of the paged-cache calls (numpy, stream by stream and head
by head) and the builder of their test inputs."""
import numpy as np

QB = 34


def half_bits_to_f64(b):
    return np.ascontiguousarray(b).view(np.float16).astype(np.float64)


def q8_to_f64(raw):
    """(..., D / 32 * 34) uint8 -> (..., D) float64."""
    b = raw.reshape(*raw.shape[:-1], -1, QB)
    d = half_bits_to_f64(b[..., :2])
    q = b[..., 2:].view(np.int8).astype(np.float64)
    return (d * q).reshape(*raw.shape[:-1], -1)


def rows_of(pool, table, n):
    """(Hkv, n, last axis) rows of one stream; pool (n_pages, Hkv, page, last axis)."""
    ps = pool.shape[2]
    if n == 0:
        return pool[0][:, :0]
    return np.concatenate([pool[p] for p in table[:-(-n // ps)]], 1)[:, :n]


def values(rows):
    return q8_to_f64(rows) if rows.dtype == np.uint8 else rows.astype(np.float64)


def scores(q, k, off, scale, causal, window, softcap):
    """q (n, D), k (len, D): (n, len) scores, -inf where unseen; `off` is the row of query 0."""
    x = q @ k.T * scale
    if softcap:
        x = softcap * np.tanh(x / softcap)
    i = np.arange(q.shape[0])[:, None] + off
    j = np.arange(k.shape[0])[None]
    see = np.ones((q.shape[0], k.shape[0]), bool)
    if causal:
        see = j <= i
        if window:
            see &= j > i - window
    return np.where(see, x, -np.inf)


def attend(c, scale=None, causal=True, window=0, softcap=0.0):
    """(out, lse, a, err) of a case: `a` = sum_j w_j |v_j| and `err` the bound on
    the f32 error of a row's scores, which the tolerances are made of."""
    D, G = c["D"], c["Hq"] // c["Hkv"]
    scale = D ** -0.5 if scale is None else scale
    T = c["q"].shape[0]
    out, a = np.zeros((2, T, c["Hq"], D))
    lse, err, tiny = np.full((T, c["Hq"]), -np.inf), np.zeros((T, c["Hq"])), np.zeros((T, c["Hq"], D))
    for s in range(len(c["len"])):
        t0, t1, n = c["start"][s], c["start"][s + 1], c["len"][s]
        if t0 == t1 or n == 0:
            continue
        kr, vr = (values(rows_of(c[p], c["table"][s], n)) for p in ("k_pool", "v_pool"))
        for h in range(c["Hq"]):
            q, k, v = c["q"][t0:t1, h].astype(np.float64), kr[h // G], vr[h // G]
            x = scores(q, k, n - (t1 - t0), scale, causal, window, softcap)
            top = x.max(1, keepdims=True)
            top = np.where(np.isinf(top), 0.0, top)
            p = np.exp(x - top)
            tot = p.sum(1, keepdims=True)
            w = p / np.where(tot > 0, tot, 1)
            out[t0:t1, h] = w @ v
            a[t0:t1, h] = w @ np.abs(v)
            tiny[t0:t1, h] = (p > 0).astype(float) @ np.abs(v) / np.where(tot > 0, tot, 1)
            with np.errstate(divide="ignore"):
                lse[t0:t1, h] = (top + np.log(tot))[:, 0]
            # f32 products and sums of D terms, the scale and the tanh
            err[t0:t1, h] = (D + 8) * 2.0 ** -24 * scale * (np.abs(q) @ np.abs(k).T).max(1, initial=0)
    return out, lse, a, err, tiny


def attend_tolerance(ref, n_half, k_half_dim=0):
    """Elementwise bounds (out in f32, lse).  n_half operands of P V are rounded
    to half (2^-11 each: P, and V where it was Q8_0); an exponential's error is
    below 2^-18, half P below 2^-14 loses at most 2^-25 of the row's largest.
    k_half_dim = D: K was rounded to half too, each product off by 2^-11."""
    out, lse, a, err, tiny = ref
    if k_half_dim:
        err = err + err / ((k_half_dim + 8) * 2.0 ** -24) * 2.0 ** -11
    fin = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    return (a * (n_half * 2.0 ** -11 + 2 * err[..., None] + 2.0 ** -17) + tiny * 2.0 ** -25 + 1e-30,
            err + 2.0 ** -18 + fin * 2.0 ** -22)


def score(c, lse, score, cap, scale=None, causal=True, window=0, softcap=0.0, observe=0, decay=1.0):
    """(new score, bound) as float64 arrays (n_seq, Hkv, cap)."""
    D, G = c["D"], c["Hq"] // c["Hkv"]
    scale = D ** -0.5 if scale is None else scale
    out, tol = score.astype(np.float64).copy(), np.zeros(score.shape)
    for s in range(len(c["len"])):
        t0, t1, n = c["start"][s], c["start"][s + 1], c["len"][s]
        out[s, :, :n] = decay * score[s, :, :n].astype(np.float64) if decay else 0.0
        o = min(t1 - t0, observe) if observe else t1 - t0
        if n == 0 or o == 0:
            continue
        kr = values(rows_of(c["k_pool"], c["table"][s], n))
        for h in range(c["Hq"]):
            q = c["q"][t0:t1, h].astype(np.float64)
            x = scores(q, kr[h // G], n - (t1 - t0), scale, causal, window, softcap)[t1 - t0 - o:]
            ls = lse[t1 - o:t1, h].astype(np.float64)[:, None]
            with np.errstate(invalid="ignore"):
                p = np.where(np.isneginf(ls) | np.isneginf(x), 0.0, np.exp(x - ls))
            # relative error of a weight: the score's f32 error, and three roundings of its exponent
            e = (D + 8) * 2.0 ** -24 * scale * (np.abs(q[t1 - t0 - o:]) @ np.abs(kr[h // G]).T)
            e = e + 2.0 ** -20 * (1 + np.where(np.isinf(x), 0, np.abs(x)) + np.abs(np.where(np.isinf(ls), 0, ls)))
            out[s, h // G, :n] += p.sum(0)
            tol[s, h // G, :n] += (p * e).sum(0)
    return out, tol + np.abs(out) * 2.0 ** -20 + 1e-30


def evict(c, sc, keep, n_sink=0, n_recent=0, row_pos=None, next_pos=None):
    """Per (stream, head): the old row of every new row; and the new lengths."""
    src, left = {}, []
    for s, n in enumerate(c["len"]):
        m = min(n, keep)
        left.append(m)
        for h in range(c["Hkv"]):
            pos = np.arange(n) if row_pos is None else row_pos[s, h, :n]
            recent = (n if next_pos is None else next_pos[s]) - n_recent
            safe = (pos < n_sink) | (pos >= recent)
            v = sc[s, h, :n].astype(np.float64)
            v = np.where(np.isnan(v), -np.inf, v)
            order = sorted(range(n), key=lambda j: (not safe[j], 0.0 if safe[j] else -v[j], j))
            kept = np.zeros(n, bool)
            kept[order[:m]] = True
            new = np.arange(m)
            new[~kept[:m]] = m + np.flatnonzero(kept[m:])
            src[s, h] = new
    return src, left


def rope(x, pos, base):
    """(T, H, D) float64, adjacent pairs rotated."""
    D = x.shape[-1]
    th = pos.astype(np.float64)[:, None] * float(np.float32(base)) ** (-2.0 * np.arange(D // 2) / D)
    c, s = np.cos(th)[:, None], np.sin(th)[:, None]
    x = x.astype(np.float64)
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return y


def build(seed, kv, streams, Hq=8, Hkv=2, D=128, page=16, poison=True, spare=3):
    """A case with streams = [(new tokens, kv_len)]: pools in shuffled pages; rows
    at or behind kv_len, spare pages and unused table entries hold poison."""
    import vtx_cases  # noqa: F401  (the package's path)
    import oracle as O
    rng = np.random.default_rng(seed)
    new, length = [x[0] for x in streams], [x[1] for x in streams]
    pages = [-(-n // page) for n in length]
    n_pages, most = sum(pages) + spare, max(max(pages), 1) + 1
    order = rng.permutation(n_pages)
    table = np.full((len(streams), most), 2 ** 31 - 1 if poison else 0, np.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    live = np.zeros((n_pages, page), bool)
    for s, n in enumerate(length):
        for r in range(n):
            live[table[s, r // page], r % page] = True
    c = {"D": D, "Hq": Hq, "Hkv": Hkv, "page": page, "kv": kv, "len": length, "table": table,
         "start": np.concatenate([[0], np.cumsum(new)]).astype(np.int32)}
    for name in ("k_pool", "v_pool"):
        x = rng.standard_normal((n_pages, Hkv, page, D)).astype(np.float32)
        if name == "k_pool":
            x *= np.where(rng.random((n_pages, Hkv, page, 1)) < 0.05, 3, 1)
        if kv == "f16":
            y = x.astype(np.float16)
            if poison:
                y[~live.repeat(Hkv, 0).reshape(n_pages, Hkv, page)] = rng.choice([np.nan, np.inf, -np.inf])
        else:
            y = O.quantize_q8_0(x)
            if poison:                       # scales of NaN
                y[~live.repeat(Hkv, 0).reshape(n_pages, Hkv, page)] = 0xff
        c[name] = y
    c["q"] = rng.standard_normal((int(c["start"][-1]), Hq, D)).astype(np.float16)
    return c
