"""Measured cases of the token-probability operators: log-probabilities of given tokens (with the
entropy and the top alternatives of each row), their gradient, and distillation from a teacher's top
logits, forward and forward + backward in one call.

``own`` selects what ``run`` computes with: False, elementary torch operations in f32; True, the
kernels of ``harp_b200`` as a program calls them (``compile_ast`` once, ``execute`` per pass)."""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_IDT = {"i32": torch.int32, "i64": torch.int64}
_BASE = {"k": 0, "dtype": "bf16", "ids": "i32", "pad": 0, "temp": 1.0, "masked": False, "entropy": False, "teacher": "f32"}


def listed():
    return [
        # one decoded token: its log-probability and the 20 alternatives an API returns
        dict(_BASE, name="logprob decode", op="logprob", n=1, v=32000, k=20),
        # a decode batch under a grammar that forbids most of the vocabulary, at temperature 0.7
        dict(_BASE, name="logprob batch masked", op="logprob", n=64, v=131072, k=20, dtype="f32", temp=0.7, masked=True),
        # prompt scoring with alternatives; an odd vocabulary, so no two rows share an alignment
        dict(_BASE, name="logprob prompt odd", op="logprob", n=2048, v=65521, k=5),
        # log-probabilities of a whole training batch (policy gradient, evaluation), no alternatives
        dict(_BASE, name="logprob batch large", op="logprob", n=4096, v=131072, ids="i64"),
        # a ten-class classifier over a batch of 65536: the label's log-probability and the best three classes
        dict(_BASE, name="logprob classes", op="logprob", n=65536, v=10, k=3, dtype="f32"),
        # gradient of a small head: launch latency
        dict(_BASE, name="gradient small", op="logprob_grad", n=32, v=1000, dtype="f32"),
        # gradient of a large batch with an entropy bonus
        dict(_BASE, name="gradient large", op="logprob_grad", n=4096, v=131072, entropy=True),
        # f16 rows inside a wider buffer, odd width and odd pitch
        dict(_BASE, name="gradient odd pitch", op="logprob_grad", n=1023, v=50021, dtype="f16", pad=28),
        # evaluating a student against stored teacher logits
        dict(_BASE, name="distill eval", op="distill", n=512, v=65536, k=64),
        # a training step of a few rows, f32
        dict(_BASE, name="distill train small", op="distill_grad", n=16, v=32000, k=8, dtype="f32"),
        # a training step at temperature 2 over an odd vocabulary, teacher logits kept in bf16
        dict(_BASE, name="distill train odd", op="distill_grad", n=1000, v=100003, k=32, temp=2.0, teacher="bf16"),
        # the largest: loss and logits gradient of a whole batch
        dict(_BASE, name="distill train large", op="distill_grad", n=4096, v=131072, k=64),
    ]


def draw(rng):
    op = rng.choice(["logprob", "logprob_grad", "distill", "distill_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    size = 4 if dtype == "f32" else 2
    while True:
        v = int(2 ** rng.uniform(1, 17.6))
        n = int(2 ** rng.uniform(0, 13))
        pad = rng.choice([0, 0, rng.randrange(1, 130)])
        if n * (v + pad) * size <= 1 << 30:
            break
    k = 0
    if op == "logprob":
        k = rng.choice([0, min(v, int(2 ** rng.uniform(0, 5)))])
    elif op != "logprob_grad":
        k = min(v, int(2 ** rng.uniform(0, 7)))
    return {"op": op, "n": n, "v": v, "k": k, "dtype": dtype, "ids": rng.choice(["i32", "i64"]), "pad": pad,
            "temp": rng.choice([1.0, round(rng.uniform(0.5, 3.0), 3)]), "masked": rng.random() < 0.25,
            "entropy": op == "logprob_grad" and rng.random() < 0.5, "teacher": rng.choice(["f32", "bf16"])}


def work(case):
    n, v, k = case["n"], case["v"], case["k"]
    size = 4 if case["dtype"] == "f32" else 2
    idb = 4 if case["ids"] == "i32" else 8
    op = case["op"]
    if op == "logprob":          # logits and ids in; logp, lse, entropy and the alternatives out
        return {"bytes": n * v * size + n * idb + 12 * n + 8 * n * k, "flops": 5 * n * v}
    if op == "logprob_grad":     # logits, ids and the row vectors in; the gradient out
        return {"bytes": 2 * n * v * size + n * idb + 4 * n * (4 if case["entropy"] else 2), "flops": 5 * n * v}
    teacher = n * k * ((4 if case["teacher"] == "f32" else 2) + idb)
    if op == "distill":
        return {"bytes": n * v * size + teacher + 4 * n, "flops": 4 * n * v}
    return {"bytes": 2 * n * v * size + teacher + 8 * n, "flops": 7 * n * v}


# ---- inputs ---------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case.  Logits are spread like a language model's: a broad bulk and, in each row, a
    few likely tokens above it; every eighth row's token is padding (-1)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, v, k = case["n"], case["v"], case["k"]
    dt, idt = _DT[case["dtype"]], _IDT[case["ids"]]
    rnd = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    z = torch.randn(n, v + case["pad"], generator=g, device="cuda").mul_(2.5)
    likely = torch.randint(0, v, (n, 8), generator=g, device="cuda")
    z.scatter_reduce_(1, likely, rnd(n, 8) * 12.0 + 4.0, "amax")
    rows = torch.arange(n, device="cuda")
    if case["masked"]:           # three quarters of the tokens forbidden, another set in each block of columns
        z.masked_fill_((rnd(1, v + case["pad"]) < 0.75).logical_and_(torch.arange(v + case["pad"], device="cuda") != likely[0, 0]), -math.inf)
    s = {"case": case, "z": z.to(dt)}
    del z
    ids = torch.where(rnd(n) < 0.5, likely[:, 0], torch.randint(0, v, (n,), generator=g, device="cuda"))
    ids = torch.where((rows % 8 == 7) & (n > 8), -1, ids)
    if case["op"] == "logprob":
        s["ids"] = ids.to(idt)
    elif case["op"] == "logprob_grad":
        s["ids"] = ids.to(idt)
        x = s["z"][:, :v].double() / case["temp"]
        lse = torch.logsumexp(x, 1)
        s["lse"] = lse.float()   # what the forward pass left
        loss_scale = 1024.0 if case["dtype"] == "f16" else 1.0      # as f16 training has it
        s["g_logp"] = torch.randn(n, generator=g, device="cuda") * (loss_scale / n)
        if case["entropy"]:
            x -= lse[:, None]
            s["ent"] = -(x.exp() * x.clamp_min(-1e4)).sum(1).float()
            s["g_ent"] = torch.full((n,), 0.01 * loss_scale / n, device="cuda")
        del x
    else:
        t = s["z"][:, :v].float()
        t += torch.randn(n, v, generator=g, device="cuda")
        val, at = torch.topk(t, k, 1)
        del t
        keep = torch.arange(k, device="cuda") < torch.where(rows % 4 == 3, (k + 1) // 2, k)[:, None]     # some rows have fewer entries
        s["teacher"] = val.masked_fill(~keep, 0.0).nan_to_num(neginf=-1e4).to(_DT[case["teacher"]])
        s["tids"] = at.masked_fill(~keep, -1).to(idt)
        if case["op"] == "distill_grad":
            s["weight"] = torch.where((rows % 8 == 7) & (n > 8), 0.0, (1024.0 if case["dtype"] == "f16" else 1.0) / n).float()
    return s


class _Memory:
    """A device buffer of harp_b200 as torch sees it (zero copy)."""

    def __init__(self, buf, shape, dtype):
        kind = {torch.float32: "<f4", torch.int32: "<i4", torch.int64: "<i8"}.get(dtype, "<i2")
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind, "data": (buf.device_ptr(), False), "version": 3}


_device = None


def _program(s):
    """What a program of harp_b200 holds: its device buffers, filled, and the compiled kernel."""
    global _device
    from harp_b200 import desc as D
    from harp_b200.backend import B200BackendRegistry, B200Buffer
    reg = B200BackendRegistry()
    if _device is None:
        _device = reg.create_device(0)
    kind = {torch.float32: D.F32, torch.float16: D.F16, torch.bfloat16: D.BF16, torch.int32: D.I32, torch.int64: D.I64}

    def new(shape, dtype):
        b = B200Buffer.allocate(_device, shape, kind[dtype], zero=False)
        return b, torch.as_tensor(_Memory(b, shape, dtype), device="cuda").view(dtype)

    c = s["case"]
    n, v, k = c["n"], c["v"], c["k"]
    dt, scale, pitch = _DT[c["dtype"]], 1.0 / c["temp"], v + c["pad"]
    common = dict(dtype=kind[dt], ids_dtype=kind[_IDT[c["ids"]]], scale=scale, stride=pitch)
    f32, i32 = torch.float32, torch.int32
    if c["op"] == "logprob":
        d = D.token_logprob(n, v, k, **common)
        names, outs = ["z", "ids"], [((n,), f32)] * 3 + ([((n, k), f32), ((n, k), i32)] if k else [])
    elif c["op"] == "logprob_grad":
        d = D.token_logprob_grad(n, v, entropy=c["entropy"], **common)
        names, outs = ["z", "ids", "lse", "g_logp"] + (["ent", "g_ent"] if c["entropy"] else []), [((n, v), dt)]
    else:
        d = D.distill_topk(n, v, k, grad=c["op"] == "distill_grad", teacher_dtype=kind[_DT[c["teacher"]]], **common)
        names, outs = ["z", "teacher", "tids"], [((n,), f32)]
        if c["op"] == "distill_grad":
            names, outs = names + ["weight"], outs + [((n, v), dt)]
    torch.cuda.synchronize()
    ins = []
    for name in names:
        b, t = new(s[name].shape, s[name].dtype)
        t.copy_(s[name])
        ins.append(b)
    made = [new(*o) for o in outs]
    torch.cuda.synchronize()
    return {"kernel": reg.compile_ast(_device, d), "ins": ins, "outs": [b for b, _ in made], "views": [t for _, t in made]}


def prepare(case, seed):
    s = _inputs(dict(_BASE, **case), seed)
    if own:
        s = _program(s)
    return s


# ---- one pass -------------------------------------------------------------------------------------

def _softmax_parts(x):
    """Row maximum (0 for a row without any finite logit), exp(x - maximum) and its row sums."""
    m = x.max(1, keepdim=True).values
    m = torch.where(m == -math.inf, 0.0, m)
    e = (x - m).exp()
    return m, e, e.sum(1, keepdim=True)


def _top(z, k):
    """The k largest of each row, equal values by the lowest index: the value's order in the upper and the
    complement of the index in the lower half of one whole number."""
    b = (z.float() + 0.0).contiguous().view(torch.int32)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long() * (1 << 32) + (z.shape[1] - 1 - torch.arange(z.shape[1], device=z.device))
    return z.shape[1] - 1 - (torch.topk(key, k, 1).values & 0xFFFFFFFF)


def _plain_logprob(s, c):
    z = s["z"][:, :c["v"]]
    x = z.float() / c["temp"]
    m, e, total = _softmax_parts(x)
    log_total = total.log()
    lse = (m + log_total)[:, 0]
    empty = total[:, 0] == 0
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < c["v"])
    own_x = x.gather(1, ids.clamp(0, c["v"] - 1)[:, None])
    logp = torch.where(there, torch.where(empty, -math.inf, (own_x - m - log_total)[:, 0]), 0.0)
    entropy = torch.where(empty, 0.0, log_total[:, 0] - (e * (x - m).clamp_min(-1e4)).sum(1) / total[:, 0])
    out = [logp, lse, entropy]
    if c["k"]:
        top = _top(z, c["k"])
        out += [torch.where(empty[:, None], -math.inf, x.gather(1, top) - m - log_total), top.int()]
    return out


def _plain_logprob_grad(s, c):
    logp = s["z"][:, :c["v"]].float() / c["temp"] - s["lse"][:, None]
    p = logp.exp()
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < c["v"])
    g = torch.where(there, s["g_logp"], 0.0)[:, None]
    d = -g * p
    if c["entropy"]:
        d -= s["g_ent"][:, None] * p * (logp.clamp_min(-1e4) + s["ent"][:, None])
    d.scatter_add_(1, ids.clamp(0, c["v"] - 1)[:, None], g)
    return [(d / c["temp"]).to(s["z"].dtype)]


def _plain_distill(s, c):
    x = s["z"][:, :c["v"]].float() / c["temp"]
    ids = s["tids"].long()
    there = (ids >= 0) & (ids < c["v"])
    ids = ids.clamp(0, c["v"] - 1)
    u = torch.where(there, s["teacher"].float() / c["temp"], -math.inf)
    mu, f, ftotal = _softmax_parts(u)
    some = ftotal > 0
    q = f / torch.where(some, ftotal, 1.0)
    log_q = u - mu - torch.where(some, ftotal, 1.0).log()
    m, e, total = _softmax_parts(x)
    log_p = x.gather(1, ids) - m - total.log()
    loss = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    if c["op"] == "distill":
        return [loss]
    d = e / total * some
    d.scatter_add_(1, ids, -q)
    return [loss, (d * (s["weight"][:, None] / c["temp"])).to(s["z"].dtype)]


def run(state):
    if own:
        state["kernel"].execute(state["ins"], state["outs"])
        return state["views"]
    c = state["case"]
    return {"logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad}.get(c["op"], _plain_distill)(state, c)


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    c = dict(_BASE, **case)
    s = _inputs(c, seed)
    v = c["v"]
    x = s["z"][:, :v].double() / c["temp"]
    if c["op"] == "logprob_grad":
        x -= s["lse"].double()[:, None]                      # log p_j, from the normaliser the call is given
        ids = s["ids"].long()
        here = (torch.arange(v, device=x.device) == ids[:, None]).double()
        g = (s["g_logp"].double() * ((ids >= 0) & (ids < v)))[:, None]
        out = here.sub_(x.exp()).mul_(g)                     # d log p_t / d x_j = [j = t] - p_j
        if c["entropy"]:                                     # d H / d x_j = -p_j (log p_j + H)
            out -= s["g_ent"].double()[:, None] * torch.where(x == -math.inf, 0.0, x.exp() * (x + s["ent"].double()[:, None]))
        return [out / c["temp"]]
    lse = torch.logsumexp(x, 1)
    logp = x.sub_(lse[:, None])
    if c["op"] == "logprob":
        ids = s["ids"].long()
        there = (ids >= 0) & (ids < v)
        mine = torch.where(there, logp.gather(1, ids.clamp(0, v - 1)[:, None])[:, 0], 0.0)
        h = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)
        out = [mine, lse, h]
        return out + [torch.topk(logp, c["k"], 1).values, None] if c["k"] else out
    ids = s["tids"].long()
    u = s["teacher"].double() / c["temp"]
    u[(ids < 0) | (ids >= v)] = -math.inf
    q = torch.softmax(u, 1)
    ids = ids.clamp(0, v - 1)
    loss = (torch.special.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, ids), 0.0)).sum(1)
    if c["op"] == "distill":
        return [loss]
    target = torch.zeros_like(logp).scatter_add_(1, ids, q)
    return [loss, logp.exp_().sub_(target).mul_((s["weight"].double() / c["temp"])[:, None])]
