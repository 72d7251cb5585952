"""Operators of codebook-compressed splats: the lookup of shared attribute rows, the log probabilities of an
assignment to them, and the loss that keeps the rows in even use.

A scene of G splats keeps, instead of one attribute row per splat (the 16 x 3 spherical-harmonic coefficients, say),
a codebook of C rows of D values and a code per splat, or a few weighted codes. Codes are learned from logits [G, C].

`run` computes a pass in plain torch operations, or, where `own` is true, through the package's entry points.
"""
import math
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_MAX_ROWS = 1 << 20  # splats
_MAX_LOGITS = 1 << 28  # splats x codes


def _package():
    if "fast-mac-gsplat_b200" not in sys.path:
        sys.path.insert(0, "fast-mac-gsplat_b200")
    import torch_gsplat_bridge_fast

    return torch_gsplat_bridge_fast


# ---- cases -----------------------------------------------------------------------------------------------------
# op "lookup": rows (splats), codes, dim (values of a codebook row), bag (weighted codes of a splat; 0: one code
#   without a weight), dtype (of the codebook), out (dtype of the result), empty (share of empty codes), skew (how
#   unevenly the codes are used: code = codes * u^skew), train (with the gradients).
# op "log_probs": rows, codes, dtype, top (alternatives asked for), pad (unused values behind each row of logits),
#   masked (share of codes that are out of use, their logits -inf), train.
# op "balance": rows, codes, dtype, bag (codes chosen of a splat), pad, masked, train.
def listed():
    return [
        # One splat is edited and shown again: its degree-3 coefficients come out of a half-precision codebook.
        dict(name="lookup_one", op="lookup", rows=1, codes=4096, dim=48, bag=0, dtype="fp16", out="fp32", empty=0.0, skew=1.0, train=False),
        # A compressed scene of 2^20 splats is unpacked for a view.
        dict(name="lookup_view", op="lookup", rows=1048576, codes=4096, dim=48, bag=0, dtype="fp16", out="fp32", empty=0.0, skew=2.0, train=False),
        # Fine-tuning the codebook of that scene, codes fixed.
        dict(name="lookup_train", op="lookup", rows=1048576, codes=8192, dim=48, bag=0, dtype="fp32", out="fp32", empty=0.0, skew=2.0, train=True),
        # Soft assignment: four weighted codes a splat, degree 2, some slots empty, odd sizes, gradients of the weights.
        dict(name="lookup_mixture", op="lookup", rows=100003, codes=1000, dim=27, bag=4, dtype="bf16", out="fp32", empty=0.1, skew=3.0, train=True),
        # One new splat gets its code and the alternatives to it.
        dict(name="log_probs_one", op="log_probs", rows=1, codes=65536, dtype="bf16", top=8, pad=0, masked=0.0, train=False),
        # Learning the codes of 65,536 splats over 4,096 rows.
        dict(name="log_probs_train", op="log_probs", rows=65536, codes=4096, dtype="fp32", top=4, pad=0, masked=0.0, train=True),
        # A minibatch over a long, pruned codebook: odd sizes, padded rows, codes out of use.
        dict(name="log_probs_long", op="log_probs", rows=2047, codes=50001, dtype="fp16", top=1, pad=15, masked=0.2, train=True),
        # A whole scene over a small codebook (one stage of a residual quantiser).
        dict(name="log_probs_small", op="log_probs", rows=1048576, codes=64, dtype="bf16", top=2, pad=0, masked=0.0, train=True),
        # The smallest training step.
        dict(name="balance_few", op="balance", rows=512, codes=64, dtype="fp32", bag=1, pad=0, masked=0.0, train=True),
        # A whole scene, two codes a splat.
        dict(name="balance_train", op="balance", rows=1048576, codes=256, dtype="bf16", bag=2, pad=0, masked=0.0, train=True),
        # A long codebook of odd size, some of it out of use.
        dict(name="balance_long", op="balance", rows=16384, codes=16383, dtype="fp16", bag=4, pad=0, masked=0.1, train=True),
        # Watching the use of the codes during evaluation: the loss and the counts alone.
        dict(name="balance_eval", op="balance", rows=65536, codes=1000, dtype="fp32", bag=1, pad=0, masked=0.0, train=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["lookup", "log_probs", "balance"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.7
    if op == "lookup":
        dim = rng.choice([3, 12, 27, 48, 59, 64, _log_int(rng, 1, 256)])
        bag = rng.choice([0, 0, rng.randint(1, 8)])
        rows = _log_int(rng, 1, min(_MAX_ROWS, (48 << 20) // (dim * max(1, bag))))
        return dict(op=op, rows=rows, codes=_log_int(rng, 1, 65536), dim=dim, bag=bag, dtype=dtype,
                    out=rng.choice(["fp32", dtype]), empty=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.5), 3)]),
                    skew=round(rng.uniform(1.0, 4.0), 2), train=train)
    codes = _log_int(rng, 8, 131072)
    rows = _log_int(rng, 1, min(_MAX_ROWS, _MAX_LOGITS // (2 * codes)))
    pad = rng.choice([0, 0, rng.randint(1, 40)])
    masked = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.6), 3)]) if codes >= 32 else 0.0
    if op == "log_probs":
        return dict(op=op, rows=rows, codes=codes, dtype=dtype, top=rng.randint(0, min(16, codes)), pad=pad, masked=masked, train=train)
    return dict(op=op, rows=rows, codes=codes, dtype=dtype, bag=rng.randint(1, min(8, codes // 4)), pad=pad, masked=masked, train=train)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _logits(case, g):
    """Logits of a half-trained assignment: normal, spread 2.5, some codes out of use; a view of padded rows."""
    G, C = case["rows"], case["codes"]
    dtype = _DTYPES[case["dtype"]]
    full = torch.empty(G, C + case["pad"], dtype=dtype, device="cuda")
    full.normal_(0.0, 2.5, generator=g)
    z = full[:, :C]
    if case["masked"]:
        out = torch.rand(C, device="cuda", generator=g) < case["masked"]
        z.masked_fill_(out, -math.inf)
        if G >= 4:
            z[G // 2] = -math.inf  # a splat that no code is left for
    return z


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    G, C = case["rows"], case["codes"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    st = dict(op=case["op"], train=case["train"], C=C)
    if case["op"] == "lookup":
        D, J = case["dim"], case["bag"]
        shape = (G, J) if J else (G,)
        st["codebook"] = (0.3 * normal(C, D)).to(_DTYPES[case["dtype"]]).requires_grad_(case["train"])
        codes = (torch.rand(shape, device="cuda", generator=g) ** case["skew"] * C).to(torch.int32).clamp_(max=C - 1)
        if case["empty"]:
            codes[torch.rand(shape, device="cuda", generator=g) < case["empty"]] = -1
        # A code's place in the codebook says nothing about its use.
        place = torch.randperm(C, device="cuda", generator=g).to(torch.int32)
        st["codes"] = torch.where(codes >= 0, place[codes.clamp(min=0).long()], codes)
        st["weights"] = torch.softmax(normal(G, J), -1).requires_grad_(case["train"]) if J else None
        st["out"] = _DTYPES[case["out"]]
        st["scale"] = 1.25
        st["g_out"] = normal(G, D).to(st["out"]) if case["train"] else None
        return st
    z = _logits(case, g)
    if case["op"] == "log_probs":
        # The code in force is a draw of the assignment; every 16th splat has none.
        code = torch.randint(0, C, (G,), device="cuda", generator=g, dtype=torch.int32)
        alive = z.gather(1, code.long()[:, None])[:, 0] > -math.inf
        code = torch.where(alive, code, z.argmax(-1).to(torch.int32))
        code[5::16] = -1
        st.update(logits=z.requires_grad_(case["train"]), codes=code, top=case["top"])
        if case["train"]:
            # Gradients of the size that a loss scaler keeps them at.
            st["g_log_probs"], st["g_entropy"], st["g_top"] = normal(G), normal(G), normal(G, case["top"])
    else:
        J = case["bag"]
        code = z.topk(J, -1).indices.to(torch.int32)
        code[3::32] = -1  # splats that take no part
        if J > 1:
            code[7::32, J - 1] = -1  # a shorter choice
        st.update(logits=z.requires_grad_(case["train"]), codes=code)
        # Scaled as a loss scaler does: the gradient's values are about 1 / (rows x codes in use) of this.
        st["g_loss"] = torch.full((), G * min(C, G * J) / 16.0, device="cuda")
    return st


# ---- one pass --------------------------------------------------------------------------------------------------
def _run_own(st):
    tgb = _package()
    if st["op"] == "lookup":
        out = tgb.codebook_lookup(st["codebook"], st["codes"], st["weights"], scale=st["scale"], out_dtype=st["out"])
        if not st["train"]:
            return [out]
        leaves = [st["codebook"]] + ([st["weights"]] if st["weights"] is not None else [])
        return [out.detach(), *torch.autograd.grad(out, leaves, st["g_out"])]
    if st["op"] == "log_probs":
        r = tgb.code_log_probs(st["logits"], st["codes"], top_k=st["top"])
        out = [r.log_probs, r.entropy, r.top_log_probs, r.top_codes]
        if not st["train"]:
            return out
        grads = [st["g_log_probs"], st["g_entropy"], st["g_top"]]
        return [t.detach() for t in out] + list(torch.autograd.grad(out[:3], st["logits"], grads))
    r = tgb.code_balance_loss(st["logits"], st["codes"])
    if not st["train"]:
        return [r.loss, r.counts]
    return [r.loss.detach(), r.counts, *torch.autograd.grad(r.loss, st["logits"], st["g_loss"])]


def _plain_lookup(st):
    codes, table, weights = st["codes"], st["codebook"].float(), st["weights"]
    if weights is None:
        codes, weights = codes[:, None], torch.ones(1, device=table.device)
    some = codes >= 0
    index = codes.clamp(min=0).long()
    w = weights * some * st["scale"]
    rows = table[index]
    out = [(rows * w[..., None]).sum(-2).to(st["out"])]
    if not st["train"]:
        return out
    g = st["g_out"].float()[:, None, :]
    grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    grad.index_add_(0, index.reshape(-1), (g * w[..., None]).reshape(-1, table.shape[1]).double())
    out.append(grad.to(st["codebook"].dtype))
    if st["weights"] is not None:
        out.append((rows * g).sum(-1) * some * st["scale"])
    return out


def _plain_softmax(z):
    """Log probabilities, probabilities (0 and -inf in rows that nothing is left of), rows with something left. In 64
    bits: next to certainty log p, 1 - p and the entropy are small differences of larger values."""
    x = z.double()
    top = x.amax(-1, keepdim=True)
    some = top > -math.inf
    e = torch.exp(x - torch.where(some, top, 0.0))
    s = torch.where(some, e.sum(-1, keepdim=True), 1.0)
    y = x - torch.where(some, top, 0.0) - torch.log(s)
    return y, e / s, some


def _plain_log_probs(st):
    z, codes, k, C = st["logits"].detach(), st["codes"], st["top"], st["C"]
    y, p, some = _plain_softmax(z)
    given = codes >= 0
    index = codes.clamp(min=0).long()[:, None]
    logp = torch.where(given, y.gather(1, index)[:, 0], 0.0)
    entropy = -torch.where(p > 0, p * y, 0.0).sum(-1)
    # Largest first, ties to the lowest index: the value's order in the high half of a whole number, the place below.
    bits = (z.float() + 0.0).view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    place = torch.arange(C - 1, -1, -1, device=z.device)
    best = C - 1 - (torch.topk((order << 32) | place, k, -1).values & 0xFFFFFFFF)
    out = [logp.float(), entropy.float(), y.gather(1, best).float(), best.to(torch.int32)]
    if not st["train"]:
        return out
    gl, gh, gt = (st["g_log_probs"] * given).double(), st["g_entropy"].double(), st["g_top"].double()
    lead = (gl + gt.sum(-1))[:, None]
    d = -p * lead - gh[:, None] * torch.where(p > 0, p * (y + entropy[:, None]), 0.0)
    d.scatter_add_(1, index, gl[:, None])
    d.scatter_add_(1, best, gt)
    return out + [torch.where(some, d, 0.0).to(z.dtype)]


def _plain_balance(st):
    z, codes, C = st["logits"].detach(), st["codes"], st["C"]
    _, p, _ = _plain_softmax(z)
    some = codes >= 0
    counts = torch.zeros(C, dtype=torch.int32, device=z.device)
    counts.index_add_(0, codes.clamp(min=0).reshape(-1).long(), some.reshape(-1).to(torch.int32))
    f = counts.double() / some.sum().clamp(min=1)
    valid = some.any(-1)
    n = valid.sum().clamp(min=1)
    d = torch.where(valid, (p * f).sum(-1), 0.0)
    loss = (C * d.sum() / n).float()
    if not st["train"]:
        return [loss, counts]
    c = torch.where(valid, st["g_loss"] * C / n, 0.0)[:, None]
    return [loss, counts, (c * p * (f - d[:, None])).to(z.dtype)]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"lookup": _plain_lookup, "log_probs": _plain_log_probs, "balance": _plain_balance}[state["op"]](state)


# ---- what a pass cannot do without, and its values in 64 bits ---------------------------------------------------
def work(case):
    G, C, s = case["rows"], case["codes"], _BYTES[case["dtype"]]
    if case["op"] == "lookup":
        D, J = case["dim"], max(1, case["bag"])
        N, so = G * J, _BYTES[case["out"]]
        touched = min(C, N)
        nbytes = touched * D * s + N * 4 + G * D * so + (N * 4 if case["bag"] else 0)
        flops = 2.0 * N * D
        if case["train"]:
            nbytes += G * D * so + C * D * s + (N * 4 if case["bag"] else 0)
            flops += 2.0 * N * D * (2 if case["bag"] else 1)
        return {"bytes": float(nbytes), "flops": flops}
    nbytes, flops = float(G) * C * s, 6.0 * G * C
    if case["op"] == "log_probs":
        nbytes += G * (12 + 8 * case["top"])
        extra = G * (8 + 4 * case["top"])
    else:
        nbytes += G * case["bag"] * 4 + C * 4
        extra = 0
    if case["train"]:
        nbytes += float(G) * C * s + extra
        flops += 6.0 * G * C
    return {"bytes": nbytes, "flops": flops}


def _exact_lookup(st):
    table = st["codebook"].detach().double().requires_grad_(True)
    codes = st["codes"]
    weights = None if st["weights"] is None else st["weights"].detach().double().requires_grad_(True)
    # An empty code is a row of zeros behind the codebook.
    wide = torch.cat([table, torch.zeros_like(table[:1])])
    index = torch.where(codes < 0, table.shape[0], codes.long())
    out = wide.index_select(0, index.reshape(-1)).view(*codes.shape, -1)
    if weights is not None:
        out = torch.einsum("gj,gjd->gd", weights, out)
    out = out * st["scale"]
    if not st["train"]:
        return [out.detach()]
    leaves = [table] + ([weights] if weights is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, st["g_out"].double())]


def _exact_log_softmax(z):
    """(leaf, log probabilities, rows with something left); rows with nothing left count as even ones."""
    x = z.detach().double().requires_grad_(True)
    some = (z > -math.inf).any(-1)
    return x, torch.log_softmax(torch.where(some[:, None], x, 0.0), -1), some


def _exact_log_probs(st):
    x, lp, some = _exact_log_softmax(st["logits"])
    codes = st["codes"]
    logp = torch.where(some, lp.gather(1, codes.clamp(min=0).long()[:, None])[:, 0], -math.inf)
    logp = torch.where(codes >= 0, logp, 0.0)
    entropy = -(lp.exp() * torch.where(lp > -math.inf, lp, 0.0)).sum(-1)
    entropy = torch.where(some, entropy, 0.0)
    order = torch.argsort(st["logits"].detach(), dim=-1, descending=True, stable=True)[:, : st["top"]]
    top = torch.where(some[:, None], lp.gather(1, order), -math.inf)
    out = [logp.detach(), entropy.detach(), top.detach(), None]
    if not st["train"]:
        return out
    loss = (torch.where(some & (codes >= 0), logp, 0.0) * st["g_log_probs"].double()).sum()
    loss = loss + (entropy * st["g_entropy"].double()).sum()
    loss = loss + (torch.where(some[:, None], top, 0.0) * st["g_top"].double()).sum()
    return out + list(torch.autograd.grad(loss, x))


def _exact_balance(st):
    x, lp, some = _exact_log_softmax(st["logits"])
    codes, C = st["codes"], st["C"]
    chosen = codes[codes >= 0].long()
    f = torch.bincount(chosen, minlength=C).double() / max(1, chosen.numel())
    valid = (codes >= 0).any(-1)
    p = lp.exp() * (some & valid)[:, None]
    loss = C * (f * p.sum(0)).sum() / max(1, int(valid.sum()))
    if not st["train"]:
        return [loss.detach(), None]
    return [loss.detach(), None, *torch.autograd.grad(loss, x, st["g_loss"].double())]


def exact(case, seed):
    st = prepare(case, seed)
    return {"lookup": _exact_lookup, "log_probs": _exact_log_probs, "balance": _exact_balance}[st["op"]](st)
