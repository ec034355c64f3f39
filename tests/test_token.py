"""The token-probability operators without a GPU: the formulas of tests/token_ref.py against automatic
differentiation and differences, the planner's choices, and what it refuses."""
import ctypes as C

import numpy as np
import pytest
import torch

import token_ref as R
from harp_b200 import capi
from harp_b200 import desc as D


def query(d, sms=148):
    info = D.CKernelInfo()
    cd = d.to_c() if isinstance(d, D.KernelDesc) else d
    capi.call("eb200_kernel_query", C.byref(cd), sms, C.byref(info))
    return info


def test_formulas_against_autograd_and_differences():
    rng = np.random.default_rng(0)
    n, v, k, scale = 6, 40, 5, 0.75
    z = rng.standard_normal((n, v)) * 3
    ids = np.array([0, 39, -1, 7, 40, 3])
    gl, gh, w = rng.standard_normal(n), rng.standard_normal(n), rng.standard_normal(n)
    zt = torch.tensor(z, requires_grad=True)
    lp = torch.log_softmax(zt * scale, 1)
    there = torch.tensor((ids >= 0) & (ids < v))
    logp = torch.where(there, lp[torch.arange(n), torch.tensor(np.clip(ids, 0, v - 1))], torch.tensor(0.0, dtype=torch.float64))
    ent = -(lp.exp() * lp).sum(1)
    out, _ = R.logprob(z, ids, k, scale)
    np.testing.assert_allclose(out["logp"], logp.detach(), rtol=1e-12)
    np.testing.assert_allclose(out["entropy"], ent.detach(), rtol=1e-12)
    np.testing.assert_allclose(out["lse"], torch.logsumexp(zt * scale, 1).detach(), rtol=1e-12)
    top = torch.topk(lp, k, 1)
    assert (out["top_ids"] == top.indices.numpy()).all()
    np.testing.assert_allclose(out["top"], top.values.detach(), rtol=1e-12)
    ((logp * torch.tensor(gl)).sum() + (ent * torch.tensor(gh)).sum()).backward()
    got, _ = R.logprob_grad(z, ids, out["lse"], gl, out["entropy"], gh, scale)
    np.testing.assert_allclose(got, zt.grad, rtol=1e-9, atol=1e-12)
    t_ids = np.stack([rng.permutation(v)[:k] for _ in range(n)])
    t_ids[1, 3:] = -1
    t_ids[2, 1] = t_ids[2, 0]
    vals = rng.standard_normal((n, k))
    res, _ = R.distill(z, vals, t_ids, scale, w)
    h = 1e-6
    for i, j in ((0, t_ids[0, 0]), (1, 5), (2, t_ids[2, 0]), (5, 11)):
        zp, zm = z.copy(), z.copy()
        zp[i, j] += h
        zm[i, j] -= h
        diff = (R.distill(zp, vals, t_ids, scale)[0]["loss"][i] - R.distill(zm, vals, t_ids, scale)[0]["loss"][i]) * w[i] / (2 * h)
        assert abs(diff - res["grad"][i, j]) < 1e-8


def test_planner():
    i = query(D.token_logprob(4096, 131072, 20, D.BF16))
    assert i.impl.decode().startswith("token_logprob_bf16") and i.launches == 1 and i.scratch_bytes == 0
    assert i.algo_bytes == 4096 * (131072 * 2 + 4 + 12 + 160)
    assert query(D.token_logprob(1, 131072, 20, D.BF16)).impl.decode() == "token_logprob_bf16_cluster"
    assert query(D.token_logprob_grad(64, 1000, True, D.F16)).impl.decode().startswith("token_logprob_grad_f16")
    i = query(D.distill_topk(2048, 50001, 32, grad=True, teacher_dtype=D.BF16, ids_dtype=D.I64, stride=50008, grad_stride=50008))
    assert i.impl.decode().startswith("distill_topk_grad_f32")
    assert i.algo_bytes == 2048 * (2 * 50001 * 4 + 32 * (2 + 8) + 8)
    assert query(D.token_logprob(0, 10)).launches == 0


def changed(d, **fields):
    c = d.to_c()
    for name, val in fields.items():
        obj, *path = [c] + name.split("__")
        for p in path[:-1]:
            obj = obj[int(p)] if p.isdigit() else getattr(obj, p)
        if path[-1].isdigit():
            obj[int(path[-1])] = val
        else:
            setattr(obj, path[-1], val)
    return c


LP, GR, KD, KG = D.token_logprob(8, 100, 5), D.token_logprob_grad(8, 100, True), D.distill_topk(8, 100, 5), D.distill_topk(8, 100, 5, grad=True)


@pytest.mark.parametrize("desc,fields,status", [
    (LP, {"ndim": 2}, capi.ERR_INVALID),
    (LP, {"shape__1": 0}, capi.ERR_INVALID),
    (LP, {"shape__0": -1}, capi.ERR_INVALID),
    (LP, {"shape__2": -1}, capi.ERR_INVALID),
    (LP, {"shape__2": 101}, capi.ERR_INVALID),                     # more alternatives than tokens
    (LP, {"shape__2": 65}, capi.ERR_UNSUPPORTED),
    (LP, {"shape__0": 1 << 27}, capi.ERR_UNSUPPORTED),
    (LP, {"shape__1": 1 << 30}, capi.ERR_UNSUPPORTED),
    (LP, {"n_inputs": 3}, capi.ERR_INVALID),
    (LP, {"scalar": 0.0}, capi.ERR_INVALID),
    (LP, {"scalar": -1.0}, capi.ERR_INVALID),
    (LP, {"scalar": float("nan")}, capi.ERR_INVALID),
    (LP, {"scalar": float("inf")}, capi.ERR_INVALID),
    (LP, {"flags": 64}, capi.ERR_INVALID),
    (LP, {"inputs__0__dtype": D.I32}, capi.ERR_UNSUPPORTED),
    (LP, {"inputs__1__dtype": D.F32}, capi.ERR_UNSUPPORTED),
    (LP, {"output__dtype": D.F16}, capi.ERR_UNSUPPORTED),
    (LP, {"inputs__0__strides__0": 99}, capi.ERR_UNSUPPORTED),     # overlapping rows
    (LP, {"inputs__0__strides__0": -100}, capi.ERR_UNSUPPORTED),
    (LP, {"inputs__0__strides__1": 2}, capi.ERR_UNSUPPORTED),
    (LP, {"inputs__0__n_bounds": 1}, capi.ERR_UNSUPPORTED),
    (LP, {"inputs__0__numel": 799}, capi.ERR_BOUNDS),
    (LP, {"inputs__0__offset": 1}, capi.ERR_BOUNDS),
    (LP, {"inputs__0__offset": -1}, capi.ERR_INVALID),
    (LP, {"inputs__1__numel": 7}, capi.ERR_BOUNDS),
    (LP, {"output__numel": 7}, capi.ERR_BOUNDS),
    (GR, {"shape__2": 1}, capi.ERR_INVALID),
    (GR, {"n_inputs": 5}, capi.ERR_INVALID),
    (GR, {"output__dtype": D.BF16}, capi.ERR_UNSUPPORTED),         # the gradient has the logits' type
    (GR, {"output__numel": 799}, capi.ERR_BOUNDS),
    (GR, {"output__strides__0": 99}, capi.ERR_UNSUPPORTED),
    (GR, {"inputs__4__dtype": D.F16}, capi.ERR_UNSUPPORTED),
    (KD, {"shape__2": 0}, capi.ERR_INVALID),
    (KD, {"shape__2": 257}, capi.ERR_UNSUPPORTED),
    (KD, {"n_inputs": 4}, capi.ERR_INVALID),
    (KD, {"inputs__1__dtype": D.I32}, capi.ERR_UNSUPPORTED),
    (KD, {"inputs__2__numel": 39}, capi.ERR_BOUNDS),
    (KG, {"n_inputs": 3}, capi.ERR_INVALID),
    (KG, {"output__dtype": D.F16}, capi.ERR_UNSUPPORTED),
    (KG, {"output__offset": 1}, capi.ERR_BOUNDS),
    (KG, {"inputs__3__numel": 7}, capi.ERR_BOUNDS),
])
def test_refusals(desc, fields, status):
    query(desc)
    with pytest.raises(capi.Eb200Error) as e:
        query(changed(desc, **fields))
    assert e.value.status == status and e.value.message


STEP_OVER = D.token_logprob(8, 100, 0, stride=120)


@pytest.mark.parametrize("desc,fields", [
    (LP, {"inputs__1__strides__0": 2}),                            # tokens two elements apart
    (LP, {"inputs__1__strides__0": -1}),
    (LP, {"inputs__1__strides__1": 3}),
    (LP, {"output__strides__0": 2}),
    (GR, {"inputs__2__strides__0": 7}),
    (GR, {"inputs__3__strides__0": 4}),
    (GR, {"inputs__4__strides__0": 2}),
    (GR, {"inputs__5__strides__0": 2}),
    (KD, {"inputs__1__strides__0": 8, "inputs__1__strides__1": 1}),       # teacher rows 8 apart, 5 wide
    (KD, {"inputs__2__strides__0": 1, "inputs__2__strides__1": 8}),       # transposed
    (KD, {"inputs__1__strides__0": 5}),                            # one entry for the whole row
    (KD, {"inputs__1__strides__0": 5, "inputs__1__strides__1": 1, "inputs__1__strides__2": 1}),
    (KD, {"output__strides__0": 3}),
    (KG, {"inputs__3__strides__0": 2}),
    (LP, {"inputs__0__strides__1": 0}),                            # one logit for the whole row, rows 100 apart
    (STEP_OVER, {"inputs__0__strides__1": 0}),
    (LP, {"inputs__0__strides__2": 1}),
    (GR, {"output__strides__1": 0}),
])
def test_strides_that_would_not_be_followed_are_refused(desc, fields):
    """Operands that the kernels take as dense, described otherwise."""
    query(desc)
    with pytest.raises(capi.Eb200Error) as e:
        query(changed(desc, **fields))
    assert e.value.status == capi.ERR_UNSUPPORTED and e.value.message


@pytest.mark.parametrize("desc,fields", [
    (LP, {"inputs__1__strides__0": 1, "output__strides__0": 1}),
    (LP, {"inputs__0__strides__0": 0, "inputs__0__strides__1": 0}),
    (KD, {"inputs__1__strides__0": 5, "inputs__1__strides__1": 1, "inputs__2__strides__0": 5, "inputs__2__strides__2": 1}),
    (D.distill_topk(8, 100, 1), {"inputs__1__strides__0": 1, "inputs__1__strides__1": 1, "inputs__2__strides__0": 1}),
    (D.distill_topk(1, 100, 5), {"inputs__1__strides__0": 99, "inputs__1__strides__1": 1}),
    (D.token_logprob(8, 1), {"inputs__0__strides__1": 0}),
    (GR, {f"inputs__{i}__strides__0": 1 for i in range(1, 6)}),
    (KG, {"inputs__3__strides__0": 1}),
])
def test_dense_operands_may_say_so(desc, fields):
    query(changed(desc, **fields))
