"""EB200_K_TOKEN_LOGPROB and EB200_K_DISTILL_TOPK: every logit counted, the longer rows' kernels with several rows per
CTA, rows summed a second time among ordinary ones, NaN and infinities in every type and operand."""
import numpy as np
import pytest

import token_ref as R
from harp_b200 import capi
from harp_b200 import desc as D
from test_gpu_token import GUARD, KIND, logits, near, rows_buffer, run_logprob, store, teacher_of, tokens, upload, value

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]
ALL_NAN = {"f32": np.nan, "f16": np.nan, "bf16": 0x7FC0}
INFINITE = {"f32": np.inf, "f16": np.inf, "bf16": 0x7F80}


def run_distill(dev, registry, stored, t_stored, ids, w, kind, tkind="f32", scale=1.0, pitch=None, offset=0):
    """Loss alone, then loss and gradient in one launch."""
    n, v = stored.shape
    k = ids.shape[1]
    common = dict(dtype=KIND[kind], teacher_dtype=KIND[tkind], scale=scale, stride=pitch, offset=offset)
    ins = [rows_buffer(dev, None, stored, kind, pitch or v, offset), upload(dev, t_stored, KIND[tkind]), upload(dev, ids, D.I32)]
    loss, loss2 = upload(dev, np.full(n, GUARD), D.F32), upload(dev, np.full(n, GUARD), D.F32)
    grad = upload(dev, store(np.full(n * v, GUARD, np.float32), kind)[0], KIND[kind])
    alone = registry.compile_ast(dev, D.distill_topk(n, v, k, **common))
    alone.execute(ins, [loss])
    both = registry.compile_ast(dev, D.distill_topk(n, v, k, grad=True, **common))
    both.execute(ins + [upload(dev, w, D.F32)], [loss2, grad])
    return loss.read_vec(), loss2.read_vec(), value(grad.read_vec(), kind).reshape(n, v), (alone, both)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,v", [(1, 1000), (3, 1025), (700, 1025), (700, 2500), (3, 8191), (500, 8193), (460, 20011), (2, 70001), (1, 131072), (3, 131071)])
def test_every_logit_is_counted_once(dev, registry, kind, n, v):
    """Rows of zeros: every exponential is 2^0 = 1 and every partial sum a whole number below 2^24, so S = V exactly and
    only the logarithm rounds (two steps, 4 U relative).  One logit lost or counted twice moves ln S by 1 / V, at least
    7.6e-6; the allowance is 2.9e-6."""
    stored, _ = store(np.zeros((n, v), np.float32), kind)
    tol = 4 * R.U * np.log(v)
    assert tol < 0.5 / v
    for k in (0, 5):
        got, kern = run_logprob(dev, registry, stored, np.full(n, v - 1), k, kind, 1.0, v + 3, 1)
        near(got["lse"], np.full(n, np.log(v)), np.full(n, tol), f"lse {kern.impl}")
        near(got["logp"], np.full(n, -np.log(v)), np.full(n, tol), f"logp {kern.impl}")
        near(got["entropy"], np.full(n, np.log(v)), np.full(n, tol), f"entropy {kern.impl}")
    loss, loss2, _, kerns = run_distill(dev, registry, stored, np.zeros((n, 1), np.float32), np.zeros((n, 1), np.int32), np.ones(n, np.float32), kind, pitch=v + 3, offset=1)
    near(loss, np.full(n, np.log(v)), np.full(n, tol), f"loss {kerns[0].impl}")
    near(loss2, np.full(n, np.log(v)), np.full(n, tol), f"loss {kerns[1].impl}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,v,k", [(1000, 20011, 0), (1400, 9001, 0), (1000, 9001, 5), (500, 33000, 20)])
def test_logprob_of_several_rows_per_cta(dev, registry, kind, n, v, k):
    rng = np.random.default_rng(v + k)
    stored, z = store(logits(rng, n, v), kind)
    ids = tokens(rng, n, v)
    got, kern = run_logprob(dev, registry, stored, ids, k, kind, 0.8, v + 1, 3)
    assert "cluster" not in kern.impl and "lanes" not in kern.impl
    ref, tol = R.logprob(z, ids, k, 0.8)
    if k:
        assert (got["top_ids"] == ref["top_ids"]).all()
    for key in tol:
        near(got[key], ref[key], tol[key], f"{key} {kern.impl}")


def mixed(rng, n, v, kind):
    """Ordinary rows between rows whose maximum is far from 0: huge, only the type's lowest value, empty."""
    z = logits(rng, n, v)
    big = 1e30 if kind != "f16" else 2e4
    z[1::4] *= big
    if kind == "f16":
        z = np.clip(z, -65504, 65504)
    z[2::8, v // 3:] = -np.inf
    z[6::8] = -np.inf
    stored, val = store(z, kind)
    lowest = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": 0xFF7F}[kind]
    stored[3::4] = lowest
    stored[7::8, 1::2] = 0xFF80 if kind == "bf16" else -np.inf
    return stored, value(stored, kind)


@pytest.mark.parametrize("kind,scale", [("f32", 1.0), ("bf16", 1.0), ("f16", 1.0), ("f16", 0.003), ("f16", 0.002)])
@pytest.mark.parametrize("n,v,k", [(1000, 3001, 0), (1000, 3001, 5), (3, 70001, 0), (9, 900, 7)])
def test_logprob_of_rows_summed_again_among_others(dev, registry, kind, scale, n, v, k):
    rng = np.random.default_rng(v)
    stored, z = mixed(rng, n, v, kind)
    ids = tokens(rng, n, v)
    got, kern = run_logprob(dev, registry, stored, ids, k, kind, scale, v + 1, 5)
    ref, tol = R.logprob(z, ids, k, scale)
    if k:
        assert (got["top_ids"] == ref["top_ids"]).all()
    for key in tol:
        near(got[key], ref[key], tol[key], f"{key} {kern.impl}")


@pytest.mark.parametrize("kind,scale", [("f32", 1.0), ("bf16", 1.0), ("f16", 1.0), ("f16", 0.002)])
@pytest.mark.parametrize("n,v,k", [(1000, 3001, 6), (320, 20011, 6), (3, 70001, 9), (9, 900, 7)])
def test_distill_of_rows_summed_again_among_others(dev, registry, kind, scale, n, v, k):
    rng = np.random.default_rng(v)
    stored, z = mixed(rng, n, v, kind)
    t_stored, t_val, ids = teacher_of(rng, n, v, k, "f32")
    w = rng.standard_normal(n).astype(np.float32)
    loss, loss2, grad, kerns = run_distill(dev, registry, stored, t_stored, ids, w, kind, "f32", scale, v + 1, 5)
    want, tol = R.distill(z, t_val, ids, scale, w, kind)
    near(loss, want["loss"], tol["loss"], f"loss {kerns[0].impl}")
    near(loss2, want["loss"], tol["loss"], f"loss {kerns[1].impl}")
    near(grad, want["grad"], tol["grad"], f"gradient {kerns[1].impl}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("n,v", [(6, 40), (6, 1000), (6, 5000), (6, 70000), (600, 3000)])
def test_nan_and_inf_logits(dev, registry, kind, bad, n, v):
    """One such logit, or nothing else, makes the row's float outputs NaN and leaves the other rows alone; NaN ranks like
    -inf.  An -inf beside a NaN stays harmless."""
    rng = np.random.default_rng(1)
    stored, _ = store(logits(rng, n, v), kind)
    b = (ALL_NAN if bad == "nan" else INFINITE)[kind]
    low = 0xFF80 if kind == "bf16" else -np.inf
    stored[3, ::2] = low
    stored[2, v // 3] = b
    stored[4] = b
    stored[5] = low
    stored[5, v - 1] = b
    z = value(stored, kind)
    odd = np.zeros(n, bool)
    odd[[2, 4, 5]] = True
    ids = np.full(n, 1)
    got, kern = run_logprob(dev, registry, stored, ids, 5, kind, 1.0, v + 1, 3)
    ref, tol = R.logprob(z[~odd], ids[~odd], 5)
    for key in tol:
        assert np.isnan(got[key][odd]).all(), (key, kern.impl)
        near(got[key][~odd], ref[key], tol[key], key)
    order = np.argsort(np.where(np.isnan(z), np.inf, -z), axis=1, kind="stable")[:, :5]
    assert (got["top_ids"] == order).all()
    # the losses against them, and the gradient: NaN where the row is, exact elsewhere; weight 0 and no entries stay 0
    t_ids = np.tile(np.arange(3, dtype=np.int32), (n, 1))
    t_val = np.tile(np.array([0.5, 0.0, -1.0], np.float32), (n, 1))
    w = np.ones(n, np.float32)
    w[4] = 0
    loss, loss2, grad, kerns = run_distill(dev, registry, stored, t_val, t_ids, w, kind, pitch=v + 1, offset=3)
    assert np.isnan(loss[odd]).all() and np.isnan(loss2[odd]).all(), kerns[0].impl
    assert np.isnan(grad[[2, 5]]).all() and (grad[4] == 0).all(), kerns[1].impl
    want, tol = R.distill(z[~odd], t_val[~odd], t_ids[~odd], 1.0, w[~odd], kind)
    near(loss[~odd], want["loss"], tol["loss"], "loss")
    near(grad[~odd], want["grad"], tol["grad"], "gradient")


@pytest.mark.parametrize("tkind", KINDS)
@pytest.mark.parametrize("n,v", [(8, 40), (8, 1000), (8, 5000), (460, 3000), (3 * 8, 20011)])
def test_nan_and_inf_among_the_teachers_values(dev, registry, tkind, n, v):
    rng = np.random.default_rng(2)
    k = 6
    z = logits(rng, n, v)
    vals, t_val = store(rng.standard_normal((n, k)).astype(np.float32), tkind)
    ids = np.stack([rng.permutation(v)[:k] for _ in range(n)]).astype(np.int32)
    vals[1, 2] = ALL_NAN[tkind]
    vals[2, 5] = INFINITE[tkind]
    vals[3, 1], ids[3, 1] = ALL_NAN[tkind], -1              # not an entry
    vals[4, 0], ids[4, 0] = INFINITE[tkind], v              # nor this
    vals[5] = ALL_NAN[tkind]
    vals[6] = 0xFF80 if tkind == "bf16" else -np.inf        # no entries
    t_val = value(vals, tkind)
    odd = np.zeros(n, bool)
    odd[[1, 2, 5]] = True
    w = rng.standard_normal(n).astype(np.float32)
    loss, loss2, grad, kerns = run_distill(dev, registry, z, vals, ids, w, "f32", tkind)
    assert np.isnan(loss[odd]).all() and np.isnan(loss2[odd]).all(), kerns[0].impl
    assert all(np.isnan(grad[i][ids[i]]).any() for i in np.nonzero(odd)[0])
    clean = np.where((ids >= 0) & (ids < v), t_val, 0.0)
    want, tol = R.distill(z[~odd], clean[~odd], ids[~odd], 1.0, w[~odd])
    near(loss[~odd], want["loss"], tol["loss"], kerns[0].impl)
    near(loss2[~odd], want["loss"], tol["loss"], kerns[1].impl)
    near(grad[~odd], want["grad"], tol["grad"], kerns[1].impl)
    assert loss[6] == 0 and (grad[6] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,v", [(6, 40), (6, 257), (6, 5000), (300, 9001)])
def test_nan_in_the_token_gradient(dev, registry, kind, n, v):
    """NaN comes out where a NaN went in (the row's lse, its g_logp, a logit) and nowhere else."""
    rng = np.random.default_rng(3)
    stored, z = store(logits(rng, n, v), kind)
    ids = rng.integers(0, v, n)
    ref, _ = R.logprob(z, ids, 0)
    lse, h = ref["lse"].astype(np.float32), ref["entropy"].astype(np.float32)
    gl, gh = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    lse[1] = np.nan
    gl[2] = np.nan
    stored[3, v // 2] = ALL_NAN[kind]
    ids[4], gl[4] = -1, np.nan                              # a padding token's gradient counts as 0
    for entropy in (False, True):
        ins = [rows_buffer(dev, rng, stored, kind, v + 1, 3), upload(dev, ids, D.I32), upload(dev, lse, D.F32), upload(dev, gl, D.F32)]
        if entropy:
            ins += [upload(dev, h, D.F32), upload(dev, gh, D.F32)]
        out = upload(dev, store(np.full(n * v, GUARD, np.float32), kind)[0], KIND[kind])
        registry.compile_ast(dev, D.token_logprob_grad(n, v, entropy, KIND[kind], stride=v + 1, offset=3)).execute(ins, [out])
        got = value(out.read_vec(), kind).reshape(n, v)
        assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
        assert np.isnan(got[3]).sum() == 1 and np.isnan(got[3, v // 2])
        plain = np.ones(n, bool)
        plain[1:4] = False
        want, tol = R.logprob_grad(z[plain], ids[plain], lse[plain], np.where(ids < 0, 0, gl)[plain], h[plain] if entropy else None,
                                   gh[plain] if entropy else None, 1.0, kind)
        near(got[plain], want, tol, f"entropy {entropy}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,v,k", [(64, 1000, 3), (64, 1025, 3), (700, 2500, 0), (700, 2500, 3), (200, 5003, 0), (6, 131072, 3), (6, 131072, 0)])
def test_a_certain_token_has_probability_one(dev, registry, kind, n, v, k):
    """Rows with one possible token (a grammar's forced one): log-probability, entropy and loss are exactly 0, whatever the
    length, since nothing is added to the token's own exponential.  Rows where another token is all but impossible:
    probabilities stay at 1 or below and entropies at 0 or above."""
    rng = np.random.default_rng(v)
    x = np.full((n, v), -np.inf, np.float32)
    ids = rng.integers(0, v, n)
    x[np.arange(n), ids] = rng.uniform(-30, 30, n)
    x[1::2] = logits(rng, (n + 1) // 2, v)[:n // 2]
    x[1::2][np.arange(n // 2), ids[1::2]] = rng.uniform(40, 70, n // 2)
    stored, z = store(x, kind)
    got, kern = run_logprob(dev, registry, stored, ids, k, kind, 0.9, v + 1, 3)
    one = slice(0, None, 2)
    assert (got["logp"][one] == 0).all(), (kern.impl, got["logp"][one].min(), got["logp"][one].max())
    assert (got["entropy"][one] == 0).all(), (kern.impl, got["entropy"][one].min(), got["entropy"][one].max())
    assert (got["logp"] <= 0).all() and (got["entropy"] >= 0).all(), kern.impl
    if k:
        assert (got["top_ids"][:, 0] == ids).all()
        assert (got["top"][one, 0] == 0).all() and np.isneginf(got["top"][one, 1:]).all() and (got["top"] <= 0).all()
    ref, tol = R.logprob(z, ids, k, 0.9)
    for key in tol:
        near(got[key], ref[key], tol[key], f"{key} {kern.impl}")
    loss, loss2, grad, kerns = run_distill(dev, registry, stored, np.zeros((n, 1), np.float32), ids[:, None].astype(np.int32), np.ones(n, np.float32), kind,
                                           "f32", 0.9, v + 1, 3)
    assert (loss[one] == 0).all() and (loss2[one] == 0).all() and (loss >= 0).all() and (loss2 >= 0).all(), kerns[0].impl
    assert (grad[one] == 0).all(), kerns[1].impl


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [1.0, 0.7, 0.45, 0.9])
@pytest.mark.parametrize("n,v", [(5, 100), (5, 1000), (40, 9001)])
def test_token_gradient_of_far_rows_stays_finite(dev, registry, kind, scale, n, v):
    """Rows of nothing but a mask's lowest value, or of huge logits: their lse in 32 bits is coarser than any ln p, but a
    probability stays within [0, 1], so each gradient within scale * (|g_logp| + |g_entropy| * (1/e + |entropy|))."""
    rng = np.random.default_rng(v)
    x = logits(rng, n, v)
    stored, _ = store(x, kind)
    stored[0] = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": 0xFF7F}[kind]
    stored[1] = stored[0]
    stored[1, ::2] = 0xFF80 if kind == "bf16" else -np.inf
    stored[2] = store(np.clip(x[2] * 1e30, -65504, 65504) if kind == "f16" else x[2] * 1e30, kind)[0]
    stored[3] = store(np.where(x[3] > 0, 3e4, -3e4) if kind == "f16" else np.where(x[3] > 0, 1e38, -1e38), kind)[0]
    ids = rng.integers(0, v, n)
    got, _ = run_logprob(dev, registry, stored, ids, 0, kind, scale)
    gl, gh = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    for entropy in (False, True):
        ins = [upload(dev, stored, KIND[kind]), upload(dev, ids, D.I32), upload(dev, got["lse"], D.F32), upload(dev, gl, D.F32)]
        if entropy:
            ins += [upload(dev, got["entropy"], D.F32), upload(dev, gh, D.F32)]
        out = upload(dev, store(np.full(n * v, GUARD, np.float32), kind)[0], KIND[kind])
        kern = registry.compile_ast(dev, D.token_logprob_grad(n, v, entropy, KIND[kind], scale=scale))
        kern.execute(ins, [out])
        g = value(out.read_vec(), kind).reshape(n, v)
        bound = scale * (np.abs(gl) + (np.abs(gh) * (np.exp(-1) + np.abs(got["entropy"])) if entropy else 0)) * (1 + 2 ** -6)
        assert np.isfinite(g).all(), (kern.impl, np.nonzero(~np.isfinite(g))[0][:4])
        assert (np.abs(g) <= bound[:, None] + 2 ** -20).all(), (kern.impl, np.abs(g).max(1) / bound)


@pytest.mark.parametrize("many", [1 << 61, 1 << 62, (1 << 62) + 5, (1 << 63) - 1])
def test_more_elements_than_64_bits_of_bytes_are_refused(dev, registry, many):
    """A descriptor may name more elements than any buffer holds; their bytes wrap around 64 bits."""
    f = lambda m, t=D.F32: upload(dev, np.zeros(m), t)       # noqa: E731
    ins, outs = [f(400), f(4, D.I32)], [f(4) for _ in range(3)]
    small = [f(1), f(1, D.I32)], [f(1) for _ in range(3)]
    for which in range(3):
        d = D.token_logprob(4, 100)
        (d.inputs + [d.output])[which].numel = many
        kern = registry.compile_ast(dev, d)
        for i, o in ((ins, outs), small):
            with pytest.raises(capi.Eb200Error) as e:
                kern.execute(i, o)
            assert e.value.status == capi.ERR_BOUNDS, e.value.message
    d = D.distill_topk(4, 100, 1, grad=True)
    d.output.numel = many
    with pytest.raises(capi.Eb200Error) as e:
        registry.compile_ast(dev, d).execute([f(400), f(4), f(4, D.I32), f(4)], [f(4), f(400)])
    assert e.value.status == capi.ERR_BOUNDS, e.value.message


@pytest.mark.parametrize("temperature", [1.0, 2.0, 0.5])
@pytest.mark.parametrize("n,v,k", [(9, 700, 12), (37, 5003, 16)])
def test_alternatives_as_the_teacher_at_a_temperature(dev, registry, temperature, n, v, k):
    """A teacher's alternatives from a pass at scale 1, distilled at another temperature: the targets are the teacher's
    logits softened once."""
    rng = np.random.default_rng(5)
    teacher, student = logits(rng, n, v), logits(rng, n, v)
    got, _ = run_logprob(dev, registry, teacher, np.zeros(n, np.int64), k, "f32")
    scale = 1.0 / temperature
    w = np.full(n, 1.0 / n, np.float32)
    loss, loss2, grad, _ = run_distill(dev, registry, student, got["top"], got["top_ids"], w, "f32", "f32", scale)
    own = np.take_along_axis(teacher, got["top_ids"], 1)
    want, tol = R.distill(student, own, got["top_ids"], scale, w)
    # the values come from the kernel: each off by its own tolerance e, which moves ln q by at most 2 scale e, q by that
    # part of itself, and the loss by sum q |ln q - ln p| of it and the change of ln q itself
    slack = 2 * scale * R.logprob(teacher, np.zeros(n, np.int64), k)[1]["top"].max()
    x = student.astype(np.float64) * scale
    ln_p = np.take_along_axis(x, got["top_ids"], 1) - np.log(np.exp(x).sum(1))[:, None]
    u = own.astype(np.float64) * scale
    q = np.exp(u) / np.exp(u).sum(1, keepdims=True)
    moved = slack * (1 + (q * np.abs(np.log(q) - ln_p)).sum(1))
    near(loss, want["loss"], tol["loss"] + moved, "loss")
    near(loss2, want["loss"], tol["loss"] + moved, "loss")
    near(grad, want["grad"], tol["grad"] + slack * scale * w[:, None], "gradient")
    if temperature != 1.0:                                  # softening in both passes is another target altogether
        twice, _ = run_logprob(dev, registry, teacher, np.zeros(n, np.int64), k, "f32", scale)
        assert np.abs(run_distill(dev, registry, student, twice["top"], twice["top_ids"], w, "f32", "f32", scale)[0] - want["loss"]).min() > moved.max()
