"""The operators on next-token distributions, as they are measured: log probabilities of given tokens with
entropy and top alternatives, their gradient, distillation from a teacher's top logits (loss and gradient),
and the scoring of tokens straight from hidden states and the output head's weight.

`listed()` and `draw()` give cases, `prepare()` makes a case's inputs on the GPU, `run()` makes one pass:
with `own` false in plain 32-bit torch operations, with `own` true through the library's entry points.
`exact()` gives the results in 64 bits.
"""
import ctypes
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WORK = 32768 * 6400            # logits of the largest listed case on given logits
HEAD_WORK = 16384 * 2048 * 32000  # multiply-adds of the largest listed head product
HEAD_LOGITS = 16384 * 32000    # logits the plain form of a head product may hold


def listed():
    return [
        # one token of a decoding loop on the scaled configuration's vocabulary: latency counts
        dict(name="logprobs_decode_1x32000", op="logprobs", rows=1, vocab=32000, dtype="bf16", k=20, scale=1.0,
             masked=False, pad=0),
        # a few rows of the fp32 logits that the model's forward writes: the smallest call
        dict(name="logprobs_f32_8x6400", op="logprobs", rows=8, vocab=6400, dtype="f32", k=5, scale=0.8,
             masked=True, pad=0),
        # an odd vocabulary whose rows start off every 16-byte boundary, with a part of it masked out
        dict(name="logprobs_odd_1021x50001", op="logprobs", rows=1021, vocab=50001, dtype="bf16", k=64, scale=1.0,
             masked=True, pad=0),
        # a teacher's record of one training batch of the 26M model (16 x 2048 tokens)
        dict(name="logprobs_batch_32768x6400", op="logprobs", rows=32768, vocab=6400, dtype="bf16", k=16, scale=1.0,
             masked=False, pad=0),
        # the gradient of a policy loss with an entropy term over the same batch
        dict(name="logprobs_bwd_32768x6400", op="logprobs_backward", rows=32768, vocab=6400, dtype="bf16", scale=1.0,
             entropy=True, masked=False, pad=0),
        # the gradient of plain log probabilities on odd fp32 rows inside a wider buffer
        dict(name="logprobs_bwd_f32_509x32001", op="logprobs_backward", rows=509, vocab=32001, dtype="f32", scale=0.7,
             entropy=False, masked=True, pad=63),
        # a distillation step of the 26M model: the teacher's 16 alternatives and the hard targets
        dict(name="distill_batch_32768x6400", op="distill", rows=32768, vocab=6400, dtype="bf16", k=16, scale=0.5,
             targets=True, normalize=True, masked=False, pad=0),
        # one sequence of the scaled configuration, the teacher's recorded log probabilities taken as they are
        dict(name="distill_2048x32000", op="distill", rows=2048, vocab=32000, dtype="bf16", k=32, scale=1.0,
             targets=False, normalize=False, masked=False, pad=0),
        # few rows of a large odd vocabulary in fp32
        dict(name="distill_f32_64x262139", op="distill", rows=64, vocab=262139, dtype="f32", k=50, scale=0.5,
             targets=True, normalize=True, masked=True, pad=0),
        # one decoded token scored on the scaled configuration's head: the weight is read once
        dict(name="head_decode_1x2048x32000", op="head", rows=1, dim=2048, vocab=32000, scale=1.0),
        # a training batch of the 26M model scored without a logits buffer
        dict(name="head_batch_32768x512x6400", op="head", rows=32768, dim=512, vocab=6400, scale=1.0),
        # a batch of the scaled configuration (8 x 2048 tokens)
        dict(name="head_batch_16384x2048x32000", op="head", rows=16384, dim=2048, vocab=32000, scale=1.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_backward", "distill", "head"])
    if op == "head":
        vocab = _log_int(rng, 64, 131072)
        dim = 8 * _log_int(rng, 8, 512)
        rows = _log_int(rng, 1, max(1, min(16384, HEAD_LOGITS // vocab, HEAD_WORK // (vocab * dim))))
        return dict(op=op, rows=rows, dim=dim, vocab=vocab, scale=rng.choice([1.0, 1.0, 0.7, 1.3]))
    vocab = _log_int(rng, 64, 262144)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    rows = _log_int(rng, 1, min(32768, WORK // (2 * vocab) if dtype == "f32" else WORK // vocab))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, scale=rng.choice([1.0, 1.0, 0.5, 0.7, 1.3]),
                masked=rng.random() < 0.4, pad=rng.choice([0, 0, 8, 13]))
    if op == "logprobs":
        case["k"] = rng.choice([0, min(vocab, _log_int(rng, 1, 128))])
    elif op == "logprobs_backward":
        case["entropy"] = rng.random() < 0.6
    else:
        case["k"] = min(vocab, _log_int(rng, 1, 128))
        case["targets"] = rng.random() < 0.5
        case["normalize"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _allowed(case, gen):
    """The columns a case leaves in: all of them, or about 70 % where it masks the vocabulary."""
    keep = torch.rand(case["vocab"], device="cuda", generator=gen) < (0.7 if case.get("masked") else 2.0)
    keep[0] = True
    return keep


def _logits(case, keep, gen):
    """[rows, vocab] logits: rows of differing sharpness around a common bias of the vocabulary, masked
    columns -inf (and, where there is a mask, one row of several wholly masked)."""
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    x = torch.empty(rows, vocab + case["pad"], device="cuda", dtype=dtype)[:, :vocab]
    v = torch.randn(rows, vocab, device="cuda", generator=gen)
    v += torch.randn(1, vocab, device="cuda", generator=gen)
    v *= 0.5 + 2.5 * torch.rand(rows, 1, device="cuda", generator=gen)
    if case["masked"]:
        v.masked_fill_(~keep, -math.inf)
        if rows > 4:
            v[rows // 2] = -math.inf
    return x.copy_(v)


def _targets(rows, keep, gen):
    """Token ids among the columns left in, with every 16th row without one (-1: padding)."""
    ids = keep.nonzero()[:, 0]
    t = ids[torch.randint(0, ids.numel(), (rows,), device="cuda", generator=gen)].int()
    t[15::16] = -1
    return t


def _row_stats(x, scale):
    """Log-sum-exp and entropy of each row, fp32, a bounded number of rows at a time."""
    parts = [_softmax(part.float(), scale) for part in x.split(max(1, (1 << 27) // x.shape[1]))]
    return torch.cat([n for _, _, n in parts]), torch.cat([_entropy(logp, p) for logp, p, _ in parts])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, op = case["rows"], case["vocab"], case["op"]
    st = dict(case=case, stream=torch.cuda.current_stream().cuda_stream)

    def out(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    keep = _allowed(case, gen)
    st["targets"] = _targets(rows, keep, gen)
    if op == "head":
        dim = case["dim"]
        st["hidden"] = torch.randn(rows, dim, device="cuda", generator=gen).bfloat16()
        st["weight"] = (torch.randn(vocab, dim, device="cuda", generator=gen) * (2.5 / math.sqrt(dim))).bfloat16()
        st["logp"], st["entropy"], st["lse"] = out(rows), out(rows), out(rows)
        return st
    x = st["logits"] = _logits(case, keep, gen)
    if op == "logprobs":
        k = case["k"]
        st["logp"], st["entropy"], st["lse"] = out(rows), out(rows), out(rows)
        st["top_logp"], st["top_ids"] = out(rows, k), out(rows, k, dtype=torch.int32)
        return st
    st["d_logits"] = out(rows, vocab, dtype=x.dtype)
    if op == "logprobs_backward":
        st["lse"], st["entropy"] = _row_stats(x, case["scale"])
        st["g_logp"] = torch.randn(rows, device="cuda", generator=gen) / rows
        st["g_entropy"] = torch.randn(rows, device="cuda", generator=gen) * (0.1 / rows) if case["entropy"] else None
        return st
    k = case["k"]
    # the teacher's alternatives: ids among the columns left in (distinct where these are enough), its log
    # probabilities falling along them, lists of unequal length
    left = keep.nonzero()[:, 0]
    first = torch.randint(0, left.numel(), (rows, 1), device="cuda", generator=gen)
    ids = left[(first + torch.arange(k, device="cuda") * max(1, left.numel() // k)) % left.numel()]
    v = torch.sort(torch.randn(rows, k, device="cuda", generator=gen) * 2 - 1, dim=1, descending=True).values
    q = torch.exp(v)
    v = torch.log(q / q.sum(1, keepdim=True) * (0.7 + 0.3 * torch.rand(rows, 1, device="cuda", generator=gen)))
    used = torch.randint(max(1, k // 2), k + 1, (rows, 1), device="cuda", generator=gen)
    ids = torch.where(torch.arange(k, device="cuda") < used, ids, torch.full_like(ids, -1))
    st["teacher_ids"], st["teacher_logits"] = ids.int().contiguous(), v.contiguous()
    w = torch.ones(rows, device="cuda")
    w[7::32] = 0.0  # rows behind a sequence's end
    st["row_weight"] = w
    # the weights of a user's loss: the distillation term, the hard targets' term, the mean over rows
    st["weights"] = (0.75 / case["scale"] ** 2, 0.25 if case["targets"] else 0.0, 1.0 / rows)
    st["loss_rows"], st["loss"] = out(rows), out(1)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _softmax(x, scale):
    """log p, p and the log-sum-exp of scale * x along the rows of fp32 x; a row with nothing left has p = 0."""
    y = x * scale
    m = y.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(y - m)
    s = e.sum(1, keepdim=True)
    lse = m + torch.log(s)
    empty = s == 0
    logp = torch.where(empty, torch.full_like(y[:, :1], -math.inf), y - lse)
    return logp, e / torch.where(empty, torch.ones_like(s), s), lse[:, 0]


def _entropy(logp, p):
    return -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)


def _at(table, ids):
    """table[r, ids[r]], and 0 where the id is no column."""
    ok = (ids >= 0) & (ids < table.shape[1])
    got = table.gather(1, torch.where(ok, ids, torch.zeros_like(ids)).long()[:, None])[:, 0]
    return torch.where(ok, got, torch.zeros_like(got)), ok


def _plain_logprobs(st):
    c = st["case"]
    logp, p, lse = _softmax(st["logits"].float(), c["scale"])
    entropy = _entropy(logp, p)
    del p
    at, _ = _at(logp, st["targets"])
    got = {"logp": at, "entropy": entropy, "lse": lse}
    if c["k"]:
        order = torch.sort(st["logits"], dim=1, descending=True, stable=True).indices[:, :c["k"]]
        got["top_logp"], got["top_ids"] = logp.gather(1, order), order.int()
    return got


def _plain_backward(st):
    c = st["case"]
    x, scale, lse = st["logits"].float(), c["scale"], st["lse"][:, None]
    some = lse != -math.inf
    logp = torch.where(some, x * scale - lse, torch.full_like(x[:, :1], -math.inf))
    p = torch.exp(logp)
    ok = (st["targets"] >= 0) & (st["targets"] < c["vocab"])
    g = torch.where(ok, st["g_logp"], torch.zeros_like(st["g_logp"]))
    d = -g[:, None] * p
    d.scatter_add_(1, torch.where(ok, st["targets"], torch.zeros_like(st["targets"])).long()[:, None], g[:, None])
    if st["g_entropy"] is not None:
        inside = torch.where(p > 0, p * (logp + st["entropy"][:, None]), torch.zeros_like(p))
        d -= st["g_entropy"][:, None] * inside
    return {"d_logits": torch.where(some, d * scale, torch.zeros_like(d)).to(st["logits"].dtype)}


def _plain_distill(st):
    c = st["case"]
    x, vocab = st["logits"].float(), c["vocab"]
    kd_w, ce_w, grad_scale = st["weights"]
    logp, p, lse = _softmax(x, c["scale"])
    ids, v = st["teacher_ids"].long(), st["teacher_logits"]
    ok = (ids >= 0) & (ids < vocab)
    v = torch.where(ok, v, torch.full_like(v, -math.inf))
    logq = v
    if c["normalize"]:
        m = v.amax(1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        logq = v - (m + torch.log(torch.exp(v - m).sum(1, keepdim=True)))
    q = torch.where(ok, torch.exp(logq), torch.zeros_like(v))
    at = torch.where(ok, ids, torch.zeros_like(ids))
    terms = torch.where(q > 0, q * (logq - logp.gather(1, at)), torch.zeros_like(q))
    loss = kd_w * terms.sum(1)
    d = p * (kd_w * c["scale"] * q.sum(1, keepdim=True))
    d.scatter_add_(1, at, q * (-kd_w * c["scale"]))
    if ce_w:
        logp1, p1, _ = (logp, p, lse) if c["scale"] == 1.0 else _softmax(x, 1.0)
        hard, has = _at(logp1, st["targets"])
        loss = loss - ce_w * hard
        d += torch.where(has[:, None], p1 * ce_w, torch.zeros_like(p1))
        one = torch.where(has, torch.full_like(hard, -ce_w), torch.zeros_like(hard))
        d.scatter_add_(1, torch.where(has, st["targets"], torch.zeros_like(st["targets"])).long()[:, None], one[:, None])
    w = st["row_weight"]
    on = (w != 0) & (lse != -math.inf)  # a row with no student left, or without weight, has no part in the loss
    loss = torch.where(on, loss * w, torch.zeros_like(loss))
    d = torch.where(on[:, None], d * (w * grad_scale)[:, None], torch.zeros_like(d))
    return {"d_logits": d.to(st["logits"].dtype), "loss_rows": loss, "loss": (loss.double().sum() * grad_scale).float().view(1)}


def _plain_head(st):
    logits = st["hidden"].float() @ st["weight"].float().t()
    logp, p, lse = _softmax(logits, st["case"]["scale"])
    return {"logp": _at(logp, st["targets"])[0], "entropy": _entropy(logp, p), "lse": lse}


# ------------------------------------------------------------------------------------------------ the library's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_logprobs(st):
    from zerollm_b200 import lib
    c, x = st["case"], st["logits"]
    k = c["k"]
    lib.call("zl_token_logprobs_" + c["dtype"], x.data_ptr(), x.stride(0), st["targets"].data_ptr(), c["rows"],
             c["vocab"], c["scale"], k, st["logp"].data_ptr(), st["entropy"].data_ptr(), st["lse"].data_ptr(),
             st["top_logp"].data_ptr() if k else None, st["top_ids"].data_ptr() if k else None, st["stream"])
    got = {"logp": st["logp"], "entropy": st["entropy"], "lse": st["lse"]}
    if k:
        got["top_logp"], got["top_ids"] = st["top_logp"], st["top_ids"]
    return got


def _own_backward(st):
    from zerollm_b200 import lib
    c, x, d = st["case"], st["logits"], st["d_logits"]
    lib.call("zl_token_logprobs_backward_" + c["dtype"], x.data_ptr(), x.stride(0), st["targets"].data_ptr(),
             st["lse"].data_ptr(), st["entropy"].data_ptr(), st["g_logp"].data_ptr(), _ptr(st["g_entropy"]),
             c["rows"], c["vocab"], c["scale"], d.data_ptr(), d.stride(0), st["stream"])
    return {"d_logits": d}


def _own_distill(st):
    from zerollm_b200 import lib
    c, x, d = st["case"], st["logits"], st["d_logits"]
    kd_w, ce_w, grad_scale = st["weights"]
    if "options" not in st:  # the same from step to step
        st["options"] = lib.DistillOptions(scale=c["scale"], teacher_scale=1.0, normalize=int(c["normalize"]),
                                           distill_weight=kd_w, target_weight=ce_w, grad_scale=grad_scale)
    lib.call("zl_distill_topk_" + c["dtype"], x.data_ptr(), x.stride(0), st["teacher_ids"].data_ptr(),
             st["teacher_logits"].data_ptr(), c["k"], st["targets"].data_ptr() if ce_w else None,
             st["row_weight"].data_ptr(), ctypes.byref(st["options"]), c["rows"], c["vocab"], d.data_ptr(), d.stride(0),
             st["loss_rows"].data_ptr(), st["loss"].data_ptr(), st["stream"])
    return {"d_logits": d, "loss_rows": st["loss_rows"], "loss": st["loss"]}


def _own_head(st):
    from zerollm_b200 import lib
    c = st["case"]
    if "workspace" not in st:  # sized once for the shape, as a program that scores batch after batch keeps it
        n = lib.load().zl_linear_logprobs_workspace_floats(c["rows"], c["dim"], c["vocab"])
        st["workspace"] = torch.empty(max(1, n), device="cuda")
    lib.call("zl_linear_logprobs_bf16", st["hidden"].data_ptr(), st["weight"].data_ptr(), st["targets"].data_ptr(),
             c["rows"], c["dim"], c["vocab"], c["scale"], st["logp"].data_ptr(), st["entropy"].data_ptr(),
             st["lse"].data_ptr(), st["workspace"].data_ptr(), st["stream"])
    return {"logp": st["logp"], "entropy": st["entropy"], "lse": st["lse"]}


PLAIN = {"logprobs": _plain_logprobs, "logprobs_backward": _plain_backward, "distill": _plain_distill,
         "head": _plain_head}
OWN = {"logprobs": _own_logprobs, "logprobs_backward": _own_backward, "distill": _own_distill, "head": _own_head}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    n = rows * vocab
    if case["op"] == "head":
        dim = case["dim"]
        return {"bytes": 2 * dim * (rows + vocab) + 16 * rows, "flops": 2 * n * dim + 5 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logprobs":
        return {"bytes": n * size + 16 * rows + 8 * rows * case["k"], "flops": 5 * n}
    if case["op"] == "logprobs_backward":
        return {"bytes": 2 * n * size + 16 * rows + (4 * rows if case["entropy"] else 0), "flops": 5 * n}
    return {"bytes": 2 * n * size + 8 * rows * case["k"] + (12 if case["targets"] else 8) * rows, "flops": 6 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(x, scale):
    """log p of fp64 rows from torch's own log-softmax; rows without a finite logit are all -inf."""
    logp = torch.log_softmax(x * scale, dim=1)
    empty = (x == -math.inf).all(1, keepdim=True)
    return logp.masked_fill(empty, -math.inf), torch.logsumexp(x * scale, dim=1), empty[:, 0]


def _exact_entropy(logp):
    return torch.special.entr(logp.exp()).sum(1)


def exact(case, seed):
    st = prepare(case, seed)
    rows, vocab, op = case["rows"], case["vocab"], case["op"]
    parts, step = [], max(1, (1 << 26) // vocab)
    for r in range(0, rows, step):
        s = slice(r, min(rows, r + step))
        t = st["targets"][s].long()
        row = torch.arange(t.numel(), device="cuda")
        has = (t >= 0) & (t < vocab)
        if op == "head":
            x = st["hidden"][s].double() @ st["weight"].double().T
        else:
            x = st["logits"][s].double()
        logp, lse, empty = _exact_rows(x, case["scale"])
        if op in ("head", "logprobs"):
            at = logp[row, t.clamp(min=0)].masked_fill(~has, 0.0)
            got = {"logp": at, "entropy": _exact_entropy(logp), "lse": lse}
            if case.get("k"):
                got["top_logp"] = logp.topk(case["k"], dim=1).values
        elif op == "logprobs_backward":
            # from the saved statistics, which are inputs here
            logp = (x * case["scale"] - st["lse"][s].double()[:, None]).masked_fill(empty[:, None], -math.inf)
            p = logp.exp()
            hot = torch.zeros_like(p)
            hot[row[has], t[has]] = 1.0
            d = st["g_logp"][s].double()[:, None] * has[:, None] * (hot - p)
            if st["g_entropy"] is not None:
                h = st["entropy"][s].double()[:, None]
                d += st["g_entropy"][s].double()[:, None] * (torch.special.entr(p) - p * h)
            got = {"d_logits": (d * case["scale"]).masked_fill(empty[:, None], 0.0)}
        else:
            kd_w, ce_w, grad_scale = st["weights"]
            ids = st["teacher_ids"][s].long()
            ok = (ids >= 0) & (ids < vocab)
            v = st["teacher_logits"][s].double().masked_fill(~ok, -math.inf)
            logq = torch.log_softmax(v, dim=1) if case["normalize"] else v
            q = logq.exp()
            dense = torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0), q)
            terms = torch.special.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, ids.clamp(min=0)), 0.0)
            loss = kd_w * terms.sum(1)
            d = kd_w * case["scale"] * (logp.exp() * q.sum(1, keepdim=True) - dense)
            if ce_w:
                logp1, _, _ = _exact_rows(x, 1.0)
                hot = torch.zeros_like(x)
                hot[row[has], t[has]] = 1.0
                loss = loss - ce_w * torch.where(has, logp1[row, t.clamp(min=0)], 0.0)
                d += ce_w * has[:, None] * (logp1.exp() - hot)
            w = st["row_weight"][s].double()
            off = (w == 0) | empty
            loss = (loss * w).masked_fill(off, 0.0)
            got = {"d_logits": (d * (w * grad_scale)[:, None]).masked_fill(off[:, None], 0.0), "loss_rows": loss}
        parts.append(got)
    if op in ("logprobs_backward", "distill"):  # the largest outputs stay in the inputs' place, not twice on the card
        st.pop("logits")
    got = {key: torch.cat([p.pop(key) for p in parts]) for key in list(parts[0])}
    if op == "distill":
        got["loss"] = (got["loss_rows"].sum() * st["weights"][2]).view(1)
    if op == "logprobs" and case["k"]:
        got["top_ids"] = None
    return got
