"""Attention over an INT8 cache for one query row of one head, three times: exactly in 64 bits, the bar that the
kernel's arithmetic keeps by the 2-norm of the row, and a NumPy model of that arithmetic (digits and all), which
shows on the CPU that the bar holds for it and fails once digits are lost.

Codes kc, vc [n, hd], scales ks, vs [n], `see` [n] the keys the row may see.

The bar.  Let w_j = e^(s_j - max), u_j = w_j * vs_j, L = sum w_j, o = sum u_j vc_j / L over the visible keys.
What the kernel rounds, and how far that moves o:
* q: half a step h = 2^(E - 24), 2^E above the row's largest magnitude (2^(E - 23) for the few largest magnitudes
  that pass three digits): s_j moves by scale * ks_j times sum_d dq_d kc_jd, of variance (h^2 / 3) |kc_j|^2; o moves
  by sum_j (u_j vc_j - w_j o) ds_j / L.
* the scores' f32 steps (8 roundings of the score) and the exponential (2^-22): the same sum, each key on its own.
* u_j, half a unit of 2^-22.99 of the largest u_j in its tile of 128 keys: variance (unit^2 / 12) |vc_j|^2 / L^2;
  and 3 roundings of its own.
* sums: every tile's share T_i = |sum_j u_j vc_j| / L passes conversion, scaling (a reciprocal and an exponential,
  2^-22 each), its merge and the last division (16 * 2^-24 covers them), and up to 4 roundings for each of the
  tiles added after it, which add up like their square root.
The independent ones enter with three times their standard deviation, the last line in full.
"""
import numpy as np

TILE = 128


def exact(q, kc, ks, vc, vs, scale, see):
    """(o, bar on |got - o|) in 64 bits."""
    q, kc, ks, vc, vs = (np.asarray(a, np.float64) for a in (q, kc, ks, vc, vs))
    if not see.any():
        return np.zeros(vc.shape[1]), 0.0
    tile = np.flatnonzero(see) // TILE
    kc, ks, vc, vs = kc[see], ks[see], vc[see], vs[see]
    s = scale * ks * (kc @ q)
    w = np.exp(s - s.max())
    u, L = w * vs, w.sum()
    o = u @ vc / L
    top, e = np.frexp(np.abs(q).max())
    h = 2.0 ** (e - 24.0 + (np.rint(top * 2.0 ** 23) > 127 * 65793))
    size = np.linalg.norm(vc, axis=1)
    lean = np.linalg.norm(u[:, None] * vc - w[:, None] * o, axis=1)
    ds2 = (scale * ks * h) ** 2 / 3 * (kc ** 2).sum(1) + (8 * 2.0 ** -24 * s) ** 2 + 2.0 ** -44
    unit, shares = np.empty(len(u)), []
    for t in np.unique(tile):
        at = tile == t
        unit[at] = 2.0 ** -22.99 * u[at].max()
        shares.append(np.linalg.norm(u[at] @ vc[at]) / L)
    noise = (lean ** 2 * ds2).sum() + ((unit ** 2 / 12 + (3 * 2.0 ** -24 * u) ** 2) * size ** 2).sum()
    return o, 3 * np.sqrt(noise) / L + (16 + 4 * np.sqrt(len(shares))) * 2.0 ** -24 * sum(shares)


def model(q, kc, ks, vc, vs, scale, see, per_row=True, lose=None):
    """The kernel's arithmetic in NumPy.  per_row: the weights' unit follows the largest product that the row sees;
    False: the largest weight and the largest value scale of the tile, each for itself, hidden keys' scales too.
    lose: "q" or "w", without the lowest digits of the query or of the weights."""
    f = np.float32
    q, ks, vs = q.astype(f), ks.astype(f), vs.astype(f)
    top = np.abs(q).max()
    e = int(np.frexp(top)[1]) if top > 0 else -100
    up = 23 - e - (int(np.rint(np.ldexp(top, 23 - e))) > 127 * 65793)  # what three signed digits hold
    X = np.rint(np.ldexp(q, up)).astype(np.int64)
    if lose == "q":
        X = (X + 128) // 256 * 256
    qf = f(np.ldexp(f(1), -up)) * (f(scale) * f(1.44269504))
    x = (kc.astype(np.int64) @ X).astype(f) * (qf * ks)
    x = np.where(see, x, f(-np.inf))
    n = len(x)
    acc, total, run = np.zeros(vc.shape[1], f), f(0), f(-np.inf)
    for a in range(0, n, TILE):
        xt, vt, ct = x[a:a + TILE], vs[a:a + TILE], vc[a:a + TILE].astype(np.int64)
        t = xt.max()
        base = max(run, t)
        if base == -np.inf:
            continue
        old = f(0) if run == -np.inf else np.exp2(run - base)
        with np.errstate(under="ignore", divide="ignore"):
            if per_row:
                p = np.exp2(xt - base)
                unit = f(2.0 ** -22.998) * max((p * vt).max(), f(2.0 ** -100))
                u = p * vt / unit
                coef = unit
            else:
                p = np.exp2(xt - t) if t > -np.inf else np.zeros_like(xt)
                unit = max(vt.max(), f(2.0 ** -100)) * f(2.0 ** -23)
                u = p * vt / unit
                coef = unit * np.exp2(t - base)
                p = p * np.exp2(t - base) if t > -np.inf else p
        W = np.rint(u).astype(np.int64)
        if lose == "w":
            W = W // 256 * 256
        acc = acc * old + (W @ ct).astype(f) * f(coef)
        total = total * old + p.sum(dtype=f)
        run = base
    return np.zeros_like(acc) if total == 0 else acc / total


def history(rng, kind, n, hd):
    """(q, kc, ks, vc, vs): a query and a history of n keys as the quantiser leaves it, and what `kind` says is odd."""
    q = rng.standard_normal(hd).astype(np.float32)
    kc, vc = (np.clip(np.rint(rng.standard_normal((n, hd)) * 42), -127, 127).astype(np.int8) for _ in range(2))
    ks, vs = ((0.5 + rng.random(n)).astype(np.float32) * np.float32(3 / 127) for _ in range(2))
    size = int(kind[-1]) if kind[-1].isdigit() else 0
    like = np.clip(np.rint(q * 42), -127, 127).astype(np.int8)
    if kind == "peaked":
        q *= 4
    elif kind.startswith("sink"):  # the first key takes most of the weight and has small values
        kc[0], vs[0] = like, np.float32(0.03 * 10.0 ** -size)
        ks[0] = np.float32((np.log(n) + 2) * np.sqrt(hd)) / np.float32(like.astype(np.float32) @ q)
    elif kind.startswith("last"):  # the last key's value scale is far above the others
        vs[n - 1] *= np.float32(10.0) ** size
    elif kind.startswith("outlier"):  # a key of hardly any weight has a large value scale
        kc[n // 2] = -like
        ks[n // 2] = np.float32(12 * np.sqrt(hd)) / np.float32(like.astype(np.float32) @ q)
        vs[n // 2] *= np.float32(10.0) ** size
    return q, kc, ks, vc, vs
