"""The token-probability operators from their formulas in 64 bits, and how far f32 arithmetic may be off.

u = 2^-24 is half a step of f32.  An exponential of a logit d below the row's maximum is off by at most
3 u |d| (the subtraction, the product with the scale, the scale's own constant) + 4 u (the exponential
itself, 2^-22), a sum of terms of one sign by one u per addition a term passes through, and a stored value by
half a step of its type."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}     # what a type's smallest step, or a flushed exponential, leaves
HEADROOM = 8.0            # a thread's reference may lie this many powers of two below its largest logit


def _parts(z, scale):
    """x - max, exp of it, and the sum S, of rows z (float64); a row of -inf has S = 0."""
    x = z * np.float64(np.float32(scale))
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        d = x - np.where(np.isneginf(m), 0.0, m)
    e = np.exp(d)
    return m[:, 0], d, e, e.sum(1)


def _rel_s(d, e, s):
    """Relative error of S: every term's own, the moved references', and the additions on the way."""
    adds = min(d.shape[1] / 32, 32) + d.shape[1] / 256 + 32      # a warp on rows of at most 1024, a CTA of 256 threads on longer ones
    near = np.where(e > 0, e * np.abs(np.maximum(d, -1e4)), 0.0).sum(1) / np.where(s > 0, s, 1.0)
    return U * (3 * near + 4 + 3 * HEADROOM + 8 + adds)


def logprob(z, ids, k, scale=1.0):
    z = np.asarray(z, np.float64)
    n, v = z.shape
    m, d, e, s = _parts(z, scale)
    empty = s == 0
    safe = np.where(empty, 1.0, s)
    ln_s = np.log(safe)
    there = (ids >= 0) & (ids < v)
    at = np.clip(ids, 0, v - 1)
    d_t = d[np.arange(n), at]
    p = e / safe[:, None]
    dd = np.maximum(d, -1e4)
    rel = _rel_s(d, e, s)
    out = {"logp": np.where(there, np.where(empty, -np.inf, d_t - ln_s), 0.0), "lse": np.where(empty, -np.inf, m + ln_s),
           "entropy": np.where(empty, 0.0, ln_s - (p * dd).sum(1))}
    mean = (p * np.abs(dd)).sum(1)
    fin = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)       # noqa: E731
    tol = {"logp": rel + 3 * U * fin(d_t) + U * fin(out["logp"]) + 2 * U * np.abs(ln_s),
           "lse": rel + 3 * U * (fin(m) + np.abs(ln_s)),
           "entropy": rel + 3 * rel * mean + 6 * U * (p * dd * dd).sum(1) + 3 * U * (mean + np.abs(ln_s))}
    if k:
        order = np.argsort(np.where(np.isnan(z), np.inf, -z), axis=1, kind="stable")[:, :k]
        top_d = np.take_along_axis(d, order, 1)
        out["top"], out["top_ids"] = np.where(empty[:, None], -np.inf, top_d - ln_s[:, None]), order.astype(np.int32)
        tol["top"] = rel[:, None] + 3 * U * fin(top_d) + U * fin(out["top"]) + 2 * U * np.abs(ln_s)[:, None]
    return out, tol


def logprob_grad(z, ids, lse, g_logp, entropy=None, g_entropy=None, scale=1.0, kind="f32"):
    z = np.asarray(z, np.float64)
    n, v = z.shape
    sc = np.float64(np.float32(scale))
    there = (ids >= 0) & (ids < v)
    gl = np.where(there, g_logp, 0.0).astype(np.float64)
    ge = np.zeros(n) if g_entropy is None else g_entropy.astype(np.float64)
    h = np.zeros(n) if entropy is None else entropy.astype(np.float64)
    zero = np.isneginf(lse) | ((gl == 0) & (ge == 0))
    with np.errstate(invalid="ignore"):
        d = z * sc - lse.astype(np.float64)[:, None]
    d = np.where(zero[:, None], -1e4, np.maximum(d, -1e4))
    p = np.exp(d)
    dense = p * (gl[:, None] + ge[:, None] * (d + h[:, None]))
    hit = np.zeros((n, v))
    hit[np.arange(n), np.clip(ids, 0, v - 1)] = gl
    out = sc * (hit - dense)
    size = p * (np.abs(gl)[:, None] + np.abs(ge)[:, None] * (np.abs(d) + np.abs(h)[:, None]))
    tol = sc * (size * U * (3 * np.abs(d) + 12) + U * np.abs(hit)) + HALF_STEP[kind] * np.abs(out) * (1 + 2 ** -6) + U * np.abs(out) + TINY[kind] * (1 + np.abs(gl) + np.abs(ge))[:, None]
    out[zero] = 0.0
    return out, tol


def distill(z, values, ids, scale=1.0, weights=None, kind="f32"):
    z, values = np.asarray(z, np.float64), np.asarray(values, np.float64)
    n, v = z.shape
    k = ids.shape[1]
    sc = np.float64(np.float32(scale))
    there = (ids >= 0) & (ids < v)
    at = np.clip(ids, 0, v - 1)
    mu, ud, f, ft = _parts(np.where(there, values, -np.inf), scale)
    some = ft > 0
    q = f / np.where(some, ft, 1.0)[:, None]
    ln_q = ud - np.log(np.where(some, ft, 1.0))[:, None]
    m, d, e, s = _parts(z, scale)
    empty = s == 0
    safe = np.where(empty, 1.0, s)
    ln_s = np.log(safe)
    d_k = np.take_along_axis(d, at, 1)
    ln_p = np.where(empty[:, None], -np.inf, d_k - ln_s[:, None])
    used = q > 0
    terms = np.where(used, q * (np.where(used, ln_q, 0.0) - np.where(used, ln_p, 0.0)), 0.0)
    loss = terms.sum(1)
    fin = lambda a: np.where(np.isfinite(a) & used, np.abs(a), 0.0)    # noqa: E731
    rel = _rel_s(d, e, s)
    rel_q = U * (3 * fin(ud) + 10 + 3 * (f * fin(ud)).sum(1, keepdims=True) + 16)
    err = q * (rel_q * (fin(ln_q) + fin(ln_p)) + rel_q + 4 * U * (fin(ln_q) + fin(ud)) + rel[:, None] + 3 * U * fin(d_k) + 3 * U * np.abs(ln_s)[:, None]
               + 2 * U * (fin(ln_q) + fin(ln_p)))
    tol_loss = err.sum(1) + 16 * U * np.where(used, q * (fin(ln_q) + fin(ln_p)), 0.0).sum(1)
    out, tol = {"loss": loss}, {"loss": tol_loss}
    if weights is not None:
        w = weights.astype(np.float64)
        p = e / safe[:, None]
        target = np.zeros((n, v))
        terr = np.zeros((n, v))
        for i in range(n):
            np.add.at(target[i], at[i], np.where(there[i], q[i], 0.0))
            np.add.at(terr[i], at[i], np.where(there[i], q[i] * (rel_q[i] + 8 * U), 0.0))
        g = (w * sc)[:, None] * (p * some[:, None] - target)
        zero = (w == 0) | empty | ~some
        g[zero] = 0.0
        gt = np.abs(w * sc)[:, None] * (p * (rel[:, None] + U * (3 * np.maximum(np.abs(np.maximum(d, -1e4)), 0) + 8)) + terr) \
            + HALF_STEP[kind] * np.abs(g) * (1 + 2 ** -6) + U * np.abs(g) + TINY[kind] * (1 + np.abs(w * sc))[:, None]
        out["grad"], tol["grad"] = g, gt
    return out, tol
