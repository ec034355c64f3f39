"""EB200_K_TOKEN_LOGPROB and EB200_K_DISTILL_TOPK on the GPU against their formulas in 64 bits
(tests/token_ref.py derives the tolerances): types, row pitches and offsets, lengths from one logit up,
few and many rows, ties, masks that leave a few logits or none, padding, and the operators one after
another as a training step uses them."""
import numpy as np
import pytest

import token_ref as R
from harp_b200 import capi
from harp_b200 import desc as D
from harp_b200.backend import B200Buffer

pytestmark = pytest.mark.gpu

KIND = {"f32": D.F32, "f16": D.F16, "bf16": D.BF16}
GUARD = 7.0          # what untouched places of outputs hold


def store(x, kind):
    """float32 -> what a buffer of `kind` holds, and the value that stands for."""
    if kind == "bf16":
        b = np.where(np.isinf(x), np.where(x > 0, 0x7F80, 0xFF80), D.bf16_bits(np.where(np.isinf(x), 0, x))).astype(np.uint16)
        return b, D.bf16_value(b)
    a = x.astype(np.float16 if kind == "f16" else np.float32)
    return a, a.astype(np.float32)


def value(a, kind):
    return (D.bf16_value(a) if kind == "bf16" else a.astype(np.float32)).astype(np.float64)


def logits(rng, n, v, how="spread"):
    z = (rng.standard_normal((n, v)) * 2.5).astype(np.float32)
    if how == "peaked":
        z[np.arange(n), rng.integers(0, v, n)] += 25.0
    elif how == "ties":
        z = rng.integers(-2, 3, (n, v)).astype(np.float32)
    elif how == "equal":
        z[...] = 1.5
    elif how == "masked":
        z[rng.random((n, v)) < 0.9] = -np.inf
        z[::3] = -np.inf
        z[::3, v // 2] = 0.25                       # one logit left
        z[1::3] = -np.inf                           # none left
    elif how == "lowest":
        z[...] = np.finfo(np.float32).min
        z[1::2, v // 3:] = -np.inf
    elif how == "rising":
        z = np.broadcast_to(np.arange(v, dtype=np.float32) / 16, (n, v)).copy()
    elif how == "huge":
        z *= 1e30
    return z


def upload(dev, a, dtype):
    b = B200Buffer.allocate(dev, [max(1, a.size)], dtype)
    if a.size:
        b.write_vec(a.reshape(-1))
    return b


def rows_buffer(dev, rng, stored, kind, pitch, offset):
    """The rows `pitch` apart from `offset`, NaN around them."""
    n, v = stored.shape
    fill = store(np.array([np.nan], np.float32), "f32")[0] if kind == "f32" else (np.array([0x7FC0], np.uint16) if kind == "bf16" else np.array([np.nan], np.float16))
    host = np.full(offset + ((n - 1) * pitch + v if n else 0), fill[0], stored.dtype)
    for i in range(n):
        host[offset + i * pitch:offset + i * pitch + v] = stored[i]
    return upload(dev, host, KIND[kind])


def near(got, ref, tol, what):
    got, ref, tol = np.broadcast_arrays(np.asarray(got, np.float64), ref, tol)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - ref) <= tol) | (got == ref) | (np.isnan(got) & np.isnan(ref)))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off; first at {i}: got {got[i]!r}, formula {ref[i]!r}, allowed {tol[i]!r}")


def run_logprob(dev, registry, stored, ids, k, kind, scale=1.0, pitch=None, offset=0, wide=False):
    n, v = stored.shape
    d = D.token_logprob(n, v, k, KIND[kind], D.I64 if wide else D.I32, scale, pitch, offset)
    kern = registry.compile_ast(dev, d)
    rng = np.random.default_rng(0)
    ins = [rows_buffer(dev, rng, stored, kind, pitch or v, offset), upload(dev, ids, D.I64 if wide else D.I32)]
    outs = [upload(dev, np.full(n, GUARD), D.F32) for _ in range(3)]
    if k:
        outs += [upload(dev, np.full(n * k, GUARD), D.F32), upload(dev, np.full(n * k, 7), D.I32)]
    kern.execute(ins, outs)
    got = dict(zip(["logp", "lse", "entropy", "top", "top_ids"], [b.read_vec() for b in outs]))
    if k:
        got["top"], got["top_ids"] = got["top"].reshape(n, k), got["top_ids"].reshape(n, k)
    return got, kern


def tokens(rng, n, v):
    ids = rng.integers(0, v, n)
    ids[3::5] = -1
    ids[4::7] = v
    return ids


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (70, 10, 3), (5, 31, 31), (9, 33, 5), (4, 64, 64), (6, 257, 20), (33, 1000, 64), (2, 1025, 20),
                                   (300, 2500, 20), (7, 4099, 64), (3, 12345, 0), (2, 32000, 20), (1, 131072, 64), (64, 40000, 20), (700, 9001, 5), (2, 1200003, 9), (20, 270001, 3)])
def test_logprob(dev, registry, kind, n, v, k):
    rng = np.random.default_rng(n * 1000 + v)
    for how, scale, pitch, offset in (("spread", 1.0, None, 0), ("peaked", 0.7, v + 13, 3), ("ties", 1.3, v + 8, 8)):
        stored, z = store(logits(rng, n, v, how), kind)
        ids = tokens(rng, n, v)
        got, kern = run_logprob(dev, registry, stored, ids, k, kind, scale, pitch, offset, wide=how == "peaked")
        ref, tol = R.logprob(z, ids, k, scale)
        if k:
            assert (got["top_ids"] == ref["top_ids"]).all(), (how, kern.impl)
        for key in tol:
            near(got[key], ref[key], tol[key], f"{key} {how} {kern.impl}")
    assert kern.launches == 1


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("how", ["masked", "equal", "lowest", "rising", "huge"])
@pytest.mark.parametrize("n,v,k", [(6, 5, 5), (7, 100, 20), (5, 900, 33), (400, 3000, 20), (3, 50000, 64), (1, 131072, 20)])
def test_logprob_of_hard_rows(dev, registry, kind, how, n, v, k):
    rng = np.random.default_rng(v)
    x = logits(rng, n, v, how)
    if kind == "f16":
        x = np.where(np.isinf(x), x, np.clip(x, -65504, 65504))
    stored, z = store(x, kind)
    if kind == "bf16" and how == "lowest":       # the type's own lowest value
        stored = np.where(np.isneginf(x), 0xFF80, 0xFF7F).astype(np.uint16)
        z = D.bf16_value(stored)
    ids = tokens(rng, n, v)
    got, kern = run_logprob(dev, registry, stored, ids, k, kind, 1.0, v + 1, 5)
    ref, tol = R.logprob(z, ids, k, 1.0)
    assert (got["top_ids"] == ref["top_ids"]).all(), kern.impl
    for key in tol:
        near(got[key], ref[key], tol[key], f"{key} {how} {kern.impl}")


@pytest.mark.parametrize("v", [40, 5000, 70000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_rows_with_nan_or_inf(dev, registry, v, bad):
    rng = np.random.default_rng(1)
    z = logits(rng, 6, v)
    z[2, v // 3] = bad
    z[4, :] = bad
    got, _ = run_logprob(dev, registry, z, np.full(6, 1), 5, "f32")
    ref, tol = R.logprob(z[[0, 1, 3, 5]], np.full(4, 1), 5)
    for key in ("logp", "lse", "entropy", "top"):
        assert np.isnan(got[key][[2, 4]]).all(), key
        near(got[key][[0, 1, 3, 5]], ref[key], tol[key], key)
    assert (got["top_ids"][[0, 1, 3, 5]] == ref["top_ids"]).all()
    order = np.argsort(np.where(np.isnan(z), np.inf, -z), axis=1, kind="stable")[:, :5]
    assert (got["top_ids"] == order).all()


@pytest.mark.parametrize("v,stride", [(131072, 2048), (131072, 16384), (65536, 8), (40000, 4)])
def test_alternatives_gathered_in_few_places(dev, registry, v, stride):
    """The largest logits recur at a period, so that a few threads hold nearly all of them."""
    rng = np.random.default_rng(2)
    z = logits(rng, 3, v)
    z[:, ::stride] += 40
    z[1, 100:5000] += 60
    for kind in ("f32", "bf16"):
        stored, val = store(z, kind)
        for n in (3, 400):
            st, va = np.resize(stored, (n, v)), np.resize(val, (n, v))
            if n == 400:
                st, va = st[:, :v // 8].copy(), va[:, :v // 8].copy()
            got, _ = run_logprob(dev, registry, st, np.zeros(n, np.int64), 64, kind)
            ref, tol = R.logprob(va, np.zeros(n, np.int64), 64)
            assert (got["top_ids"] == ref["top_ids"]).all()
            near(got["top"], ref["top"], tol["top"], "top")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("n,v", [(1, 1), (5, 3), (40, 10), (7, 129), (33, 1000), (9, 4097), (2, 60001)])
def test_logprob_grad(dev, registry, kind, entropy, n, v):
    rng = np.random.default_rng(v)
    for how, scale, pitch, offset, gp, go in (("spread", 1.0, None, 0, None, 0), ("peaked", 0.5, v + 3, 1, v + 9, 2), ("masked", 1.7, v + 1, 0, v + 2, 5)):
        stored, z = store(logits(rng, n, v, how), kind)
        ids = tokens(rng, n, v)
        ref, _ = R.logprob(z, ids, 0, scale)
        lse, h = ref["lse"].astype(np.float32), ref["entropy"].astype(np.float32)
        gl, gh = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
        gl[::6] = 0
        gh[::4] = 0
        d = D.token_logprob_grad(n, v, entropy, KIND[kind], D.I32, scale, pitch, offset, gp, go)
        kern = registry.compile_ast(dev, d)
        ins = [rows_buffer(dev, rng, stored, kind, pitch or v, offset), upload(dev, ids, D.I32), upload(dev, lse, D.F32), upload(dev, gl, D.F32)]
        if entropy:
            ins += [upload(dev, h, D.F32), upload(dev, gh, D.F32)]
        guard = store(np.full(d.output.numel, GUARD, np.float32), kind)[0]
        out = upload(dev, guard, KIND[kind])
        kern.execute(ins, [out])
        got = value(out.read_vec(), kind)
        want, tol = R.logprob_grad(z, ids, lse, gl, h if entropy else None, gh if entropy else None, scale, kind)
        gp = gp or v
        touched = np.zeros(got.size, bool)
        for i in range(n):
            at = slice(go + i * gp, go + i * gp + v)
            near(got[at], want[i], tol[i], f"row {i} {how} {kern.impl}")
            touched[at] = True
        assert (got[~touched] == GUARD).all()


def teacher_of(rng, n, v, k, kind):
    ids = np.stack([rng.permutation(v)[:k] if v >= k else rng.integers(0, v, k) for _ in range(n)])
    vals = (rng.standard_normal((n, k)) * 3).astype(np.float32)
    ids[1::4, k // 2:] = -1                       # fewer entries
    ids[2::4, k // 3:] = v + 5
    vals[2::4, : k // 4] = -np.inf
    if n > 4:
        ids[4] = -1                               # none
    if k > 2:
        ids[3::5, 2] = ids[3::5, 0]               # the same index twice
    stored, val = store(vals, kind)
    return stored, val, ids


@pytest.mark.parametrize("kind,tkind", [("f32", "f32"), ("f16", "bf16"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (5, 3, 2), (6, 4, 9), (40, 10, 3), (7, 130, 32), (20, 1000, 256), (600, 1500, 16), (9, 4097, 33), (2, 60001, 64), (1, 131072, 128), (320, 20011, 8), (2, 1200003, 20), (20, 270001, 16)])
def test_distill(dev, registry, kind, tkind, n, v, k):
    rng = np.random.default_rng(v + k)
    for how, scale, pitch, offset, gp, go in (("spread", 1.0, None, 0, None, 0), ("peaked", 0.5, v + 3, 1, v + 9, 2), ("masked", 1.7, v + 1, 0, v + 2, 5)):
        stored, z = store(logits(rng, n, v, how), kind)
        t_stored, t_val, ids = teacher_of(rng, n, v, k, tkind)
        w = rng.standard_normal(n).astype(np.float32)
        w[::5] = 0
        wide = how == "peaked"
        common = dict(dtype=KIND[kind], teacher_dtype=KIND[tkind], ids_dtype=D.I64 if wide else D.I32, scale=scale, stride=pitch, offset=offset)
        ins = [rows_buffer(dev, rng, stored, kind, pitch or v, offset), upload(dev, t_stored, KIND[tkind]), upload(dev, ids, common["ids_dtype"])]
        want, tol = R.distill(z, t_val, ids, scale, w, kind)
        loss = upload(dev, np.full(n, GUARD), D.F32)
        kern = registry.compile_ast(dev, D.distill_topk(n, v, k, **common))
        kern.execute(ins, [loss])
        alone = loss.read_vec()
        near(alone, want["loss"], tol["loss"], f"loss {how} {kern.impl}")
        d = D.distill_topk(n, v, k, grad=True, grad_stride=gp, grad_offset=go, **common)
        kern = registry.compile_ast(dev, d)
        loss2 = upload(dev, np.full(n, GUARD), D.F32)
        grad = upload(dev, store(np.full(d.output.numel, GUARD, np.float32), kind)[0], KIND[kind])
        kern.execute(ins + [upload(dev, w, D.F32)], [loss2, grad])
        near(loss2.read_vec(), want["loss"], tol["loss"], f"loss {how} {kern.impl}")
        got = value(grad.read_vec(), kind)
        gp = gp or v
        touched = np.zeros(got.size, bool)
        for i in range(n):
            at = slice(go + i * gp, go + i * gp + v)
            near(got[at], want["grad"][i], tol["grad"][i], f"row {i} {how} {kern.impl}")
            touched[at] = True
        assert (got[~touched] == GUARD).all()


def test_rows_of_weight_zero_ignore_their_logits(dev, registry):
    rng = np.random.default_rng(3)
    n, v, k = 4, 3000, 4
    z = logits(rng, n, v)
    z[1] = np.nan
    ids = np.tile(np.arange(k), (n, 1))
    w = np.array([1, 0, 1, 1], np.float32)
    ins = [upload(dev, z, D.F32), upload(dev, np.zeros((n, k)), D.F32), upload(dev, ids, D.I32), upload(dev, w, D.F32)]
    loss, grad = upload(dev, np.zeros(n), D.F32), upload(dev, np.full(n * v, GUARD), D.F32)
    registry.compile_ast(dev, D.distill_topk(n, v, k, grad=True)).execute(ins, [loss, grad])
    g = grad.read_vec().reshape(n, v)
    assert (g[1] == 0).all() and np.isfinite(g).all()
    lse = np.array([0, np.nan, 0, 0], np.float32)
    ids = np.array([5, -1, 7, 9])
    ins = [upload(dev, z, D.F32), upload(dev, ids, D.I32), upload(dev, lse, D.F32), upload(dev, np.ones(n), D.F32)]
    registry.compile_ast(dev, D.token_logprob_grad(n, v)).execute(ins, [grad])
    g = grad.read_vec().reshape(n, v)
    assert (g[1] == 0).all() and np.isfinite(g).all()


def test_results_do_not_depend_on_the_run(dev, registry):
    """Bit for bit the same again, and inside a replayed graph, whatever ran in between."""
    rng = np.random.default_rng(4)
    for n, v in ((3, 70001), (500, 6007)):
        k = 20
        z = logits(rng, n, v, "ties")
        ids = rng.integers(0, v, n)
        t_ids = np.stack([rng.permutation(v)[:k] for _ in range(n)])
        zb, ib, tb, wb = upload(dev, z, D.F32), upload(dev, ids, D.I32), upload(dev, rng.standard_normal((n, k)), D.F32), upload(dev, rng.standard_normal(n), D.F32)
        tib = upload(dev, t_ids, D.I32)
        lp = registry.compile_ast(dev, D.token_logprob(n, v, k))
        kd = registry.compile_ast(dev, D.distill_topk(n, v, k, grad=True))

        def buffers():
            return [upload(dev, np.zeros(n), D.F32) for _ in range(3)] + [upload(dev, np.zeros(n * k), D.F32), upload(dev, np.zeros(n * k), D.I32)], \
                [upload(dev, np.zeros(n), D.F32), upload(dev, np.zeros(n * v), D.F32)]
        a, ag = buffers()
        b, bg = buffers()
        lp.execute([zb, ib], a)
        kd.execute([zb, tb, tib, wb], ag)
        dev.synchronize()
        dev.graph_begin()
        lp.execute([zb, ib], b)
        kd.execute([zb, tb, tib, wb], bg)
        g = dev.graph_end()
        for _ in range(3):
            g.launch()
        for x, y in zip(a + ag, b + bg):
            assert (x.read_vec() == y.read_vec()).all()


def test_the_operators_together(dev, registry):
    """A teacher's alternatives train a student: the teacher's pass returns values and indices, distillation takes
    them, and one SGD update of the student's logits lowers nothing but what its gradient says."""
    rng = np.random.default_rng(5)
    n, v, k = 37, 5003, 16
    teacher, student = logits(rng, n, v), logits(rng, n, v)
    ids = rng.integers(0, v, n)
    tz, sz, ib = upload(dev, teacher, D.F32), upload(dev, student, D.F32), upload(dev, ids, D.I32)
    stats = [upload(dev, np.zeros(n), D.F32) for _ in range(3)]
    top, top_ids = upload(dev, np.zeros(n * k), D.F32), upload(dev, np.zeros(n * k), D.I32)
    registry.compile_ast(dev, D.token_logprob(n, v, k)).execute([tz, ib], stats + [top, top_ids])
    w = np.full(n, 1.0 / n, np.float32)
    loss, grad = upload(dev, np.zeros(n), D.F32), upload(dev, np.zeros(n * v), D.F32)
    registry.compile_ast(dev, D.distill_topk(n, v, k, grad=True)).execute([sz, top, top_ids, upload(dev, w, D.F32)], [loss, grad])
    lp = registry.compile_ast(dev, D.token_logprob(n, v))
    lp.execute([sz, ib], stats)
    gl = np.full(n, -0.5 / n, np.float32)
    grad2 = upload(dev, np.zeros(n * v), D.F32)
    registry.compile_ast(dev, D.token_logprob_grad(n, v)).execute([sz, ib, stats[1], upload(dev, gl, D.F32)], [grad2])
    ref, _ = R.logprob(teacher, ids, k)
    want, tol = R.distill(student, ref["top"].astype(np.float32), ref["top_ids"], 1.0, w)
    # the teacher's values come from the kernel: off by what its own tolerance allows, which moves q by twice that
    slack = 2 * R.logprob(teacher, ids, k)[1]["top"].max()
    near(loss.read_vec(), want["loss"], tol["loss"] + slack * (1 + np.abs(want["loss"])) * 10, "loss")
    near(grad.read_vec().reshape(n, v), want["grad"], tol["grad"] + slack / n, "distillation gradient")
    s_ref, s_tol = R.logprob(student, ids, 0)
    want2, tol2 = R.logprob_grad(student, ids, stats[1].read_vec(), gl)
    near(grad2.read_vec().reshape(n, v), want2, tol2, "token gradient")
    both = grad.read_vec() + grad2.read_vec()
    # the gradient against a difference of the losses along itself (in 64 bits)
    step = 1e-4
    f = lambda z: (R.distill(z, ref["top"].astype(np.float32), ref["top_ids"])[0]["loss"] * w).sum() + (R.logprob(z, ids, 0)[0]["logp"] * gl).sum()   # noqa: E731
    g = both.reshape(n, v).astype(np.float64)
    slope = (f(student + step * g) - f(student - step * g)) / (2 * step)
    # the central difference is off by step^2 / 6 times a third derivative below |g|^3, and by rounding of f
    assert abs(slope - (g * g).sum()) <= 1e-6 * (g * g).sum() + 2.0 ** -50 * 100 / step


def test_refusals(dev, registry):
    k = registry.compile_ast(dev, D.token_logprob(4, 100, 3))
    f = lambda m, t=D.F32: upload(dev, np.zeros(m), t)       # noqa: E731
    z, ids = f(400), f(4, D.I32)
    outs = [f(4), f(4), f(4), f(12), f(12, D.I32)]

    def refused(status, ins, o):
        with pytest.raises(capi.Eb200Error) as e:
            k.execute(ins, o)
        assert e.value.status == status, e.value.message
    refused(capi.ERR_INVALID, [z, ids], outs[:3])                       # too few outputs
    refused(capi.ERR_INVALID, [z], outs)
    refused(capi.ERR_BOUNDS, [z, f(3, D.I32)], outs)
    refused(capi.ERR_BOUNDS, [f(399), ids], outs)
    refused(capi.ERR_BOUNDS, [z, ids], outs[:3] + [f(11), outs[4]])
    refused(capi.ERR_BOUNDS, [z, ids], outs[:4] + [f(11, D.I32)])
    refused(capi.ERR_INVALID, [z, ids], [outs[0], outs[0], outs[2], outs[3], outs[4]])
    refused(capi.ERR_INVALID, [z, ids], [outs[0], z, outs[2], outs[3], outs[4]])
    k.execute([z, ids], outs)                                           # and the right call still runs
    assert abs(outs[2].read_vec()[0] - np.log(100)) < 1e-5
    # no rows: nothing to do
    e = registry.compile_ast(dev, D.token_logprob(0, 100, 3))
    e.execute([f(1), f(1, D.I32)], [f(1), f(1), f(1), f(1), f(1, D.I32)])
    assert e.launches == 0
