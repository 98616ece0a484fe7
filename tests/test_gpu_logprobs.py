"""The operators on next-token distributions on the GPU, through the C ABI, against plain fp64 formulas.

Tolerances, derived from the operators' arithmetic (u = 2^-24, half a step of fp32):
  * one exponential e^(y - y_max): its argument is off by 2u |y - y_max| (a difference and a product, in
    powers of two), the exponential itself by 2^-22: relative (4 + 2 |y - y_max|) u.  Weighted with
    e^-|y - y_max| the argument's part is at most 2u / e.
  * S0 and S1 are sums of at most n = ceil(vocab / (256 * vector)) * vector + 16 terms per thread and 16 joins:
    relative (n + 16 + 6) u at worst, each join another rounding of 2^-22: 16 * 4u.
    ERR = (n + 100) u covers both.
  * lse = y_max + ln S0 and ln p = (x - x_max) scale - ln S0: ERR + 4u (|y - y_max| + ln vocab + |y_max|).
  * H = ln S0 - S1 / S0: ERR (1 + |S1 / S0|) + 4u (ln vocab + 1), S1 / S0 <= ln vocab + 1.
  * a gradient entry: relative error of p times its factors (each a few u), one rounding to the output's type.
    A p below the least normal number 2^-126 counts as 0: at most FLUSH times p's factor more, where a factor
    |ln p| is at most 88 at 2^-126 (and p |ln p| falls below it).
"""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLUSH = 2.0 ** -126
NINF = -math.inf
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def L():
    from zerollm_b200 import lib
    lib.load()
    return lib


def stream():
    return torch.cuda.current_stream().cuda_stream


def err(vocab, dtype):
    vec = 8 if dtype == "bf16" else 4
    return (math.ceil(vocab / (256 * vec)) * vec + 116) * U


def half_step(dtype):
    return 2.0 ** -8 if dtype == "bf16" else U


def ptr(t):
    return None if t is None else t.data_ptr()


def strided(rows, vocab, dtype, pad=0, offset=0):
    """[rows, vocab] in rows of vocab + pad elements, `offset` elements into an allocation filled with a sentinel."""
    buf = torch.full((rows * (vocab + pad) + offset + 64,), 7.0, device="cuda", dtype=DT[dtype])
    return torch.as_strided(buf, (rows, vocab), (vocab + pad, 1), offset), buf


def make(kind, rows, vocab, dtype, pad=0, offset=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + rows * 131 + vocab)
    x, _ = strided(rows, vocab, dtype, pad, offset)
    v = torch.randn(rows, vocab, device="cuda", generator=g) * 3
    if kind == "masked":
        v.masked_fill_(torch.rand(vocab, device="cuda", generator=g) < 0.4, NINF)
        v[:, 0] = 1.0
        v[rows // 2] = NINF                                   # a row with nothing left
    elif kind == "few":                                       # constrained decoding: a handful allowed
        keep = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        keep[torch.randperm(vocab, device="cuda", generator=g)[:5]] = True
        v.masked_fill_(~keep, NINF)
    elif kind == "lowest":                                    # masked with the type's lowest value
        low = torch.finfo(DT[dtype]).min
        v.masked_fill_(torch.rand(vocab, device="cuda", generator=g) < 0.4, low)
        v[rows // 2] = low
        v[:, 0] = torch.where(v[:, 0] == low, v[:, 0], v[:, 0])
    elif kind == "highest":                                   # one token forced with the type's highest value
        v[:, vocab // 3] = torch.finfo(DT[dtype]).max
    elif kind == "constant":
        v.fill_(-2.5)
    elif kind == "ties":                                      # few distinct values, both zeros among them
        v = torch.randint(-2, 3, (rows, vocab), device="cuda", generator=g).float() * 0.5
        v[:, 1::2] = torch.where(v[:, 1::2] == 0, -torch.zeros_like(v[:, 1::2]), v[:, 1::2])
    elif kind == "sorted":
        v = v.sort(dim=1).values
    elif kind == "sharp":
        v = v * 10
    elif kind == "column":                                    # the largest all in one thread's elements
        vec = 8 if dtype == "bf16" else 4
        v[:, ::256 * vec] += 40
        for j in range(1, vec):
            v[:, j::256 * vec] += 40
    else:
        assert kind == "normal"
    x.copy_(v)
    return x


def softmax64(x, scale):
    """ln p, lse of fp64 rows by the definition; a row with nothing left is -inf."""
    y = x.double() * scale
    m = y.amax(1, keepdim=True)
    m = torch.where(m == NINF, torch.zeros_like(m), m)
    ln_s = torch.log(torch.exp(y - m).sum(1, keepdim=True))   # kept apart from m, which may be -3.4e38
    logp = torch.where(ln_s == NINF, torch.full_like(y[:, :1], NINF), y - m - ln_s)
    return logp, (m + ln_s)[:, 0]


def entropy64(logp):
    p = logp.exp()
    return -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, device=got.device, dtype=torch.float64).expand_as(got)
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got)), f"{what}: finite places differ"
    assert torch.equal(got[~fin], want[~fin]), f"{what}: infinities differ"
    d = (got - want).abs()[fin]
    assert bool((d <= tol[fin]).all()), f"{what}: off by {float((d / tol[fin].clamp(min=1e-300)).max()):.3g} x tolerance, {float(d.max()):.3g}"


def targets_for(rows, vocab, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 5)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[0] = vocab - 1
    if rows > 2:
        t[1], t[2] = -1, vocab                               # padding and one past the end
    return t


def call_logprobs(L, x, dtype, targets, scale, k, st=None):
    rows, vocab = x.shape
    out = {n: torch.full((rows,), 7.0, device="cuda") for n in ("logp", "entropy", "lse")}
    top = torch.full((rows, k), 7.0, device="cuda")
    ids = torch.full((rows, k), -7, device="cuda", dtype=torch.int32)
    L.call(f"zl_token_logprobs_{dtype}", x.data_ptr(), x.stride(0), ptr(targets), rows, vocab, scale, k,
           out["logp"].data_ptr() if targets is not None else None, out["entropy"].data_ptr(), out["lse"].data_ptr(),
           top.data_ptr() if k else None, ids.data_ptr() if k else None, st if st is not None else stream())
    return out, top, ids


def check_logprobs(L, x, dtype, scale, k, targets):
    rows, vocab = x.shape
    scale = C.c_float(scale).value
    out, top, ids = call_logprobs(L, x, dtype, targets, scale, k)
    torch.cuda.synchronize()
    logp, lse = softmax64(x, scale)
    E, lnv = err(vocab, dtype), math.log(vocab)
    ymax = torch.where(lse == NINF, torch.zeros_like(lse), (x.double() * scale).amax(1))
    tol_row = E + 4 * U * (lnv + ymax.abs())
    close(out["lse"], lse, tol_row, "lse")
    close(out["entropy"], entropy64(logp), E * (2 + lnv) + 4 * U * (lnv + 1), "entropy")
    if targets is not None:
        ok = (targets >= 0) & (targets < vocab)
        at = logp.gather(1, targets.clamp(0, vocab - 1).long()[:, None])[:, 0]
        want = torch.where(ok, at, torch.zeros_like(at))
        away = torch.where(torch.isfinite(at), at.abs(), torch.zeros_like(at))
        close(out["logp"], want, E + 4 * U * (lnv + away), "logp")
    if k:
        order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(ids.long(), order), "top ids"
        at = logp.gather(1, order)
        away = torch.where(torch.isfinite(at), at.abs(), torch.zeros_like(at))
        close(top, at, E + 4 * U * (lnv + away), "top_logp")


SIZES = [(1, 1), (3, 2), (2, 7), (5, 31), (4, 64), (3, 257), (6, 1000), (2, 2048), (3, 4099), (5, 6400), (2, 8193),
         (300, 640), (1, 32000), (2, 50001), (400, 20001), (1, 150001),
         (1200, 3), (1301, 100), (1200, 2049), (5000, 130), (1250, 6401), (1190, 16000), (1184, 30000), (1300, 40000)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_token_logprobs_sizes(L, rows, vocab, dtype):
    x = make("normal", rows, vocab, dtype)
    for k in sorted({0, 1, min(vocab, 20), min(vocab, 128)}):
        check_logprobs(L, x, dtype, 1.0, k, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["masked", "few", "lowest", "highest", "constant", "ties", "sorted", "sharp", "column"])
@pytest.mark.parametrize("rows,vocab,k", [(3, 900, 20), (3, 6400, 16), (7, 6400, 128), (1, 33333, 50), (2, 140000, 64),
                                          (1200, 900, 20), (1201, 6400, 64), (2500, 5003, 1),
                                          (1500, 130, 100), (1300, 300, 64), (1200, 1024, 128), (5, 1023, 97), (600, 1100, 20)])
def test_token_logprobs_values(L, rows, vocab, k, kind, dtype):
    check_logprobs(L, make(kind, rows, vocab, dtype), dtype, 1.0, k, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset,scale", [(0, 1, 1.0), (8, 0, 0.7), (13, 3, 1.3), (1, 5, 0.25)])
def test_token_logprobs_strides(L, pad, offset, scale, dtype):
    for rows, vocab in [(4, 6), (5, 1001), (3, 6400), (2, 20000), (1300, 1001)]:
        check_logprobs(L, make("normal", rows, vocab, dtype, pad, offset), dtype, scale, min(vocab, 9), targets_for(rows, vocab))


def test_token_logprobs_nan_and_inf_rows(L):
    """A NaN or +inf logit spoils its own row's statistics and no other; the ids stay distinct columns."""
    x = make("normal", 4, 700, "f32")
    x[1, 33] = math.nan
    x[2, 44] = math.inf
    out, top, ids = call_logprobs(L, x, "f32", targets_for(4, 700), 1.0, 8)
    for n in ("entropy", "lse"):
        assert torch.isnan(out[n][1]) and torch.isnan(out[n][2]) and torch.isfinite(out[n][[0, 3]]).all()
    assert int(ids[2, 0]) == 44 and 33 not in ids[1].tolist()
    for r in range(4):
        got = ids[r].tolist()
        assert len(set(got)) == 8 and min(got) >= 0 and max(got) < 700
    x[1] = math.nan  # nothing but NaN: the lowest indices
    _, _, ids = call_logprobs(L, x, "f32", targets_for(4, 700), 1.0, 8)
    assert ids[1].tolist() == list(range(8))


@pytest.mark.parametrize("rows,vocab,k", [(1500, 150, 100), (1500, 300, 64), (1500, 1001, 128)])
def test_token_logprobs_nan_in_short_rows(L, rows, vocab, k):
    """NaN logits come last among the alternatives, by their index."""
    x = make("normal", rows, vocab, "bf16")
    x[1] = math.nan
    x[2, k // 2:] = math.nan
    x[3] = -math.inf
    x[3, 5] = math.nan
    out, _, ids = call_logprobs(L, x, "bf16", targets_for(rows, vocab), 1.0, k)
    assert ids[1].tolist() == list(range(k))
    assert sorted(ids[2, :k // 2].tolist()) == list(range(k // 2)) and ids[2, k // 2:].tolist() == list(range(k // 2, k))
    assert ids[3].tolist() == [i for i in range(k + 1) if i != 5]
    assert torch.isfinite(out["lse"][torch.arange(rows, device="cuda") > 3]).all() and torch.isnan(out["lse"][1:3]).all()


def test_token_logprobs_optional_outputs(L):
    x = make("normal", 3, 500, "bf16")
    out, _, ids = call_logprobs(L, x, "bf16", targets_for(3, 500), 1.0, 4)
    ids2 = torch.empty_like(ids)
    L.call("zl_token_logprobs_bf16", x.data_ptr(), 500, None, 3, 500, 1.0, 4, None, None, None, None, ids2.data_ptr(), stream())
    assert torch.equal(ids, ids2)
    logp = torch.empty(3, device="cuda")
    t = targets_for(3, 500)
    L.call("zl_token_logprobs_bf16", x.data_ptr(), 500, t.data_ptr(), 3, 500, 1.0, 0, logp.data_ptr(), None, None, None, None, stream())
    assert torch.equal(logp, out["logp"])


# ------------------------------------------------------------------ gradient of the log probabilities
def call_backward(L, x, dtype, t, lse, ent, gl, ge, scale, d):
    rows, vocab = x.shape
    L.call(f"zl_token_logprobs_backward_{dtype}", x.data_ptr(), x.stride(0), ptr(t), lse.data_ptr(), ptr(ent), ptr(gl),
           ptr(ge), rows, vocab, scale, d.data_ptr(), d.stride(0), stream())


def backward64(x, t, lse, ent, gl, ge, scale):
    rows, vocab = x.shape
    none = (lse.abs() > 1e30)[:, None]   # rows masked wholly, or with a token forced by the type's highest value
    logp = torch.where(none, torch.full((), NINF, device="cuda", dtype=torch.float64), x.double() * scale - lse.double()[:, None])
    p = logp.exp()
    g = torch.zeros(rows, device="cuda", dtype=torch.float64) if gl is None else gl.double()
    g = torch.where((t >= 0) & (t < vocab), g, torch.zeros_like(g)) if t is not None else g
    hot = torch.zeros_like(p)
    if t is not None:
        ok = ((t >= 0) & (t < vocab)).nonzero()[:, 0]
        hot[ok, t[ok].long()] = 1
    h = torch.zeros_like(g) if ge is None else ge.double()
    H = torch.zeros_like(g) if ent is None else ent.double()
    l0 = torch.where(p > 0, logp, torch.zeros_like(p))
    d = scale * (g[:, None] * (hot - p) - h[:, None] * p * (l0 + H[:, None]))
    size = scale * (g.abs()[:, None] * (hot + p) + h.abs()[:, None] * p * (l0.abs() + H.abs()[:, None]))
    # p: argument l off by 2u (|l| + |lse|) and 2^-22 of the exponential; the products a few u
    tol = size * (4 * (l0.abs() + torch.where(none[:, 0], torch.zeros_like(lse), lse).abs().double()[:, None]) + 12) * U
    tol = tol + FLUSH * scale * (g.abs() + h.abs() * (88 + H.abs()))[:, None]
    return torch.where(none, torch.zeros_like(d), d), torch.where(none, torch.zeros_like(tol), tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,pad,offset,dpad,kind", [
    (1, 1, 0, 0, 0, "normal"), (3, 7, 0, 1, 0, "normal"), (5, 257, 3, 0, 3, "normal"), (3, 6400, 0, 0, 0, "masked"),
    (4, 6401, 0, 0, 0, "normal"), (3, 6400, 13, 0, 0, "normal"), (3, 5003, 13, 2, 5, "masked"), (2, 40001, 0, 0, 0, "sharp"),
    (3, 2000, 0, 0, 0, "few"), (3, 2000, 0, 0, 0, "lowest"), (3, 2000, 0, 0, 0, "highest")])
@pytest.mark.parametrize("which", ["logp", "entropy", "both"])
def test_token_logprobs_backward(L, rows, vocab, pad, offset, dpad, kind, dtype, which):
    scale = C.c_float(0.7).value
    x = make(kind, rows, vocab, dtype, pad, offset)
    t = targets_for(rows, vocab)
    out, _, _ = call_logprobs(L, x, dtype, t, scale, 0)
    g = torch.Generator(device="cuda").manual_seed(4)
    gl = torch.randn(rows, device="cuda", generator=g) if which != "entropy" else None
    ge = torch.randn(rows, device="cuda", generator=g) if which != "logp" else None
    ent = out["entropy"] if ge is not None else None
    d, buf = strided(rows, vocab, dtype, dpad, 0)
    call_backward(L, x, dtype, t, out["lse"], ent, gl, ge, scale, d)
    want, tol = backward64(x, t, out["lse"], ent, gl, ge, scale)
    close(d, want, tol + half_step(dtype) * (want.abs() + tol) + FLUSH, "d_logits")
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, d.shape, d.stride(), 0).fill_(False)
    assert bool((buf[mask] == 7.0).all()), "wrote outside its rows"
    if pad == 0:  # in the logits' place
        y = x.clone()
        call_backward(L, y, dtype, t, out["lse"], ent, gl, ge, scale, y)
        assert torch.equal(y, d)


def test_token_logprobs_gradient_by_differences(L):
    """The gradient against central differences of the forward: step h, rounding of the summed loss ~ 40 u / h
    per difference and a third-order term h^2 / 6 times a bounded derivative (|f'''| <= 8 for these weights)."""
    rows, vocab, scale, h = 2, 37, 1.0, 0.03
    x = make("normal", rows, vocab, "f32")
    t = torch.tensor([3, 36], device="cuda", dtype=torch.int32)
    gl = torch.tensor([0.7, -1.1], device="cuda")
    ge = torch.tensor([0.5, 0.9], device="cuda")

    def f(z):
        o, _, _ = call_logprobs(L, z, "f32", t, scale, 0)
        return gl.double() * o["logp"].double() + ge.double() * o["entropy"].double()

    o, _, _ = call_logprobs(L, x, "f32", t, scale, 0)
    d = torch.empty_like(x)
    call_backward(L, x, "f32", t, o["lse"], o["entropy"], gl, ge, scale, d)
    tol = 8 * h * h / 6 + 200 * U / h
    for j in range(vocab):
        a, b = x.clone(), x.clone()
        a[:, j] += h
        b[:, j] -= h
        step = (a[:, j] - b[:, j]).double()
        diff = (f(a) - f(b)) / step
        assert float((diff - d[:, j].double()).abs().max()) < tol


# ------------------------------------------------------------------ distillation
def teacher(rows, vocab, k, seed=0, dup=False, columns=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 11)
    pool = torch.arange(vocab, device="cuda") if columns is None else columns
    ids = torch.stack([pool[torch.randperm(pool.numel(), device="cuda", generator=g)[torch.arange(k, device="cuda") % pool.numel()]]
                       for _ in range(rows)]).int() if k else torch.empty(rows, 0, device="cuda", dtype=torch.int32)
    v = torch.randn(rows, k, device="cuda", generator=g) - 3.0
    if dup and k > 3:
        ids[:, 3] = ids[:, 0]
    if rows > 1 and k:
        ids[1, k // 2:] = -1                               # a short list
    if rows > 2 and k:
        ids[2] = vocab                                     # no alternative at all
    if k > 4:
        v[0, 4] = NINF
    return ids.contiguous(), v.contiguous()


def distill64(x, ids, v, t, w, o):
    rows, vocab = x.shape
    logp, lse = softmax64(x, o.scale)
    logp1, _ = softmax64(x, 1.0)
    ok = (ids >= 0) & (ids < vocab)
    y = torch.where(ok, v.double() * o.teacher_scale, torch.full((), NINF, device="cuda", dtype=torch.float64))
    ln_n = torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
    if o.normalize and ids.shape[1]:
        ln_n = torch.logsumexp(y, 1, keepdim=True)
        ln_n = torch.where(ln_n == NINF, torch.zeros_like(ln_n), ln_n)
    lq = y - ln_n
    q = torch.where(ok, lq.exp(), torch.zeros_like(lq))
    at = ids.clamp(0, vocab - 1).long()
    lp = logp.gather(1, at)
    ent = torch.where(q > 0, q * lq, torch.zeros_like(q))
    crs = torch.where(q > 0, -q * lp, torch.zeros_like(q))
    kd, ce = o.distill_weight, o.target_weight
    loss = (kd * (ent + crs)).sum(1) if kd else torch.zeros(rows, device="cuda", dtype=torch.float64)
    sq = q.sum(1, keepdim=True)
    dense = torch.zeros_like(logp).scatter_add_(1, at, q)
    p, p1 = logp.exp(), logp1.exp()
    d = kd * o.scale * (p * sq - dense)
    size = abs(kd) * o.scale * (p * sq + dense)
    away = abs(kd) * (ent.abs() + torch.where(torch.isfinite(crs), crs.abs(), torch.zeros_like(crs))).sum(1)
    if ce:
        has = (t >= 0) & (t < vocab)
        tt = t.clamp(0, vocab - 1).long()[:, None]
        hard = torch.where(has, logp1.gather(1, tt)[:, 0], torch.zeros_like(loss))
        loss = loss - ce * hard
        hot = torch.zeros_like(p).scatter_(1, tt, 1.0) * has[:, None]
        d = d + ce * (torch.where(has[:, None], p1, torch.zeros_like(p1)) - hot)
        size = size + abs(ce) * (p1 + hot)
        away = away + abs(ce) * torch.where(torch.isfinite(hard), hard.abs(), torch.zeros_like(hard))
    w = torch.ones(rows, device="cuda") if w is None else w
    off = (w == 0) | (lse == NINF)
    loss = torch.where(off, torch.zeros_like(loss), loss * w)
    f = (w * o.grad_scale).double()[:, None]
    d = torch.where(off[:, None], torch.zeros_like(d), d * f)
    size = size * f.abs()
    return loss, d, size, FLUSH * (abs(kd) * o.scale * sq + abs(ce)) * f.abs(), (abs(kd) * (1 + sq[:, 0]) + abs(ce), away * w.abs())


def check_distill(L, x, dtype, k, o, targets=True, weights=True, dup=False, dpad=0, columns=None):
    rows, vocab = x.shape
    ids, v = teacher(rows, vocab, k, dup=dup, columns=columns)
    t = targets_for(rows, vocab) if targets else None
    if columns is not None and t is not None:
        t[0] = int(columns[0])
    w = None
    if weights:
        w = torch.linspace(0.5, 1.5, rows, device="cuda")
        if rows > 3:
            w[3] = 0.0
            x[3, :5] = math.nan                             # a row of no weight may hold anything
    d, buf = strided(rows, vocab, dtype, dpad, 0)
    lr, lo = torch.full((rows,), 7.0, device="cuda"), torch.full((1,), 7.0, device="cuda")

    def go(x, d, lr, lo):
        L.call(f"zl_distill_topk_{dtype}", x.data_ptr(), x.stride(0), ids.data_ptr() if k else None, v.data_ptr() if k else None,
               k, ptr(t), ptr(w), C.byref(o), rows, vocab, ptr(d), d.stride(0) if d is not None else 0, lr.data_ptr(), ptr(lo), stream())

    go(x, d, lr, lo)
    clean = x.clone()
    if weights and rows > 3:
        clean[3, :5] = 0
    loss, want, size, flush, (weight, away) = distill64(clean, ids, v, t, w, o)
    E, lnv = err(vocab, dtype), math.log(vocab) + 1
    loss = torch.where(loss > torch.finfo(torch.float32).max, torch.full_like(loss, math.inf), loss)  # (beyond an fp32 output)
    # each ln p is off by E + 4u (ln vocab + |ln p|), each q by 8u |ln q| + 132 u (its sum); products of both
    close(lr, loss, 2 * weight * E + 4 * U * lnv * weight + 160 * U * away * 4 + 1e-30, "loss_rows")
    if torch.isfinite(loss).all():
        tot = loss.sum() * o.grad_scale
        slack = ((2 * weight * E + 4 * U * lnv * weight + 640 * U * away).sum() * abs(o.grad_scale))
        assert abs(float(lo) - float(tot)) <= float(slack) + 2 * U * abs(float(tot)) + 1e-30
    spread = (clean.double() * o.scale)
    spread = torch.where(torch.isfinite(spread), spread, torch.zeros_like(spread))
    tol = size * (E + (160 + 8 * math.log(max(2, vocab))) * U + 4 * U * (spread - spread.amax(1, keepdim=True)).abs().clamp(max=200))
    close(d, want, tol + half_step(dtype) * (want.abs() + tol) + flush + FLUSH, "d_logits")
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, d.shape, d.stride(), 0).fill_(False)
    assert bool((buf[mask] == 7.0).all()), "wrote outside its rows"
    lr2 = torch.empty_like(lr)
    go(x, None, lr2, None)                                  # the loss alone
    assert torch.equal(lr2, lr)
    if x.is_contiguous() and dpad == 0:                     # (at the same place within 16 bytes: the same order of sums)
        y, _ = strided(rows, vocab, dtype, 0, x.data_ptr() % 16 // x.element_size())
        y.copy_(x)
        go(y, y, lr2, lo)                                   # the gradient in the logits' place
        assert torch.equal(y, d) and torch.equal(lr2, lr)


def opts(L, scale=1.0, teacher_scale=1.0, normalize=1, kd=0.75, ce=0.25, gs=0.125):
    f = lambda a: C.c_float(a).value  # noqa: E731
    return L.DistillOptions(f(scale), f(teacher_scale), normalize, f(kd), f(ce), f(gs))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (4, 7, 3), (5, 257, 20), (4, 6400, 16), (5, 6401, 128), (1, 33333, 50),
                                          (4, 50001, 64), (400, 1000, 5), (2, 140000, 32), (3, 6400, 0)])
def test_distill_sizes(L, rows, vocab, k, dtype):
    check_distill(L, make("normal", rows, vocab, dtype), dtype, k, opts(L))
    check_distill(L, make("normal", rows, vocab, dtype), dtype, k, opts(L, scale=0.5, teacher_scale=0.5, ce=1.5), dup=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("o", [dict(normalize=0), dict(kd=0.0), dict(ce=0.0), dict(ce=0.0, scale=0.3), dict(kd=0.0, scale=2.0),
                               dict(scale=2.0, teacher_scale=3.0, normalize=0, gs=-3.0), dict(gs=0.0),
                               dict(scale=0.25), dict(scale=0.5, kd=0.0)])
@pytest.mark.parametrize("targets,weights", [(True, True), (True, False)])
def test_distill_options(L, o, targets, weights, dtype):
    check_distill(L, make("normal", 5, 3001, dtype), dtype, 17, opts(L, **o), targets, weights, dup=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["masked", "few", "lowest", "highest", "constant", "sharp"])
@pytest.mark.parametrize("vocab", [900, 6400, 40001])
def test_distill_values(L, kind, vocab, dtype):
    x = make(kind, 5, vocab, dtype)
    columns = torch.isfinite(x[0].float()).nonzero()[:, 0] if kind in ("masked", "few") else None
    check_distill(L, x, dtype, 12, opts(L, scale=0.7), columns=columns)
    check_distill(L, make(kind, 5, vocab, dtype), dtype, 12, opts(L, scale=0.7))   # alternatives the student has masked


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset,dpad", [(0, 1, 0), (13, 0, 0), (0, 0, 13), (8, 3, 8), (13, 5, 2)])
def test_distill_strides(L, pad, offset, dpad, dtype):
    for rows, vocab in [(4, 9), (5, 1001), (4, 20000)]:
        check_distill(L, make("normal", rows, vocab, dtype, pad, offset), dtype, min(vocab, 6), opts(L, scale=0.8), dpad=dpad)


def test_distill_gradient_by_differences(L):
    """d_logits against central differences of loss_out (third-order and rounding terms as above; |f'''| <= 8)."""
    rows, vocab, k, h = 2, 29, 6, 0.03
    o = opts(L, scale=0.8, teacher_scale=0.9, gs=0.5)
    x = make("normal", rows, vocab, "f32")
    ids, v = teacher(rows, vocab, k, dup=True)
    t = torch.tensor([4, 28], device="cuda", dtype=torch.int32)
    lr, lo, d = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)

    def f(z, d=None):
        L.call("zl_distill_topk_f32", z.data_ptr(), vocab, ids.data_ptr(), v.data_ptr(), k, t.data_ptr(), None, C.byref(o),
               rows, vocab, ptr(d), vocab, lr.data_ptr(), lo.data_ptr(), stream())
        return lr.double() * o.grad_scale

    f(x, d)
    tol = 8 * h * h / 6 + 200 * U / h
    for j in range(vocab):
        a, b = x.clone(), x.clone()
        a[:, j] += h
        b[:, j] -= h
        step = (a[:, j] - b[:, j]).double()
        assert float(((f(a) - f(b)) / step - d[:, j].double()).abs().max()) < tol


# ------------------------------------------------------------------ together, and how they are called
def test_record_then_distill(L):
    """A teacher's record written by the first operator trains a student by the third: with the student equal to
    the teacher and all of the vocabulary recorded the loss is 0 and so is the gradient."""
    rows, vocab = 6, 100
    x = make("normal", rows, vocab, "f32")
    out, top, ids = call_logprobs(L, x, "f32", targets_for(rows, vocab), 1.0, vocab)
    lr, lo, d = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)
    o = opts(L, normalize=0, kd=1.0, ce=0.0, gs=1.0)
    L.call("zl_distill_topk_f32", x.data_ptr(), vocab, ids.data_ptr(), top.data_ptr(), vocab, None, None, C.byref(o), rows, vocab,
           d.data_ptr(), vocab, lr.data_ptr(), lo.data_ptr(), stream())
    # q and p agree to E + 40u relative each: sum q (ln q - ln p) <= their difference, and so is each gradient entry
    tol = 2 * (err(vocab, "f32") + 160 * U * (1 + math.log(vocab)))
    assert float(lr.abs().max()) < tol and float(d.abs().max()) < tol
    # and the plain cross-entropy's gradient is the log probabilities' gradient with g = -1
    t = targets_for(rows, vocab)
    o = opts(L, kd=0.0, ce=1.0, gs=1.0)
    L.call("zl_distill_topk_f32", x.data_ptr(), vocab, None, None, 0, t.data_ptr(), None, C.byref(o), rows, vocab, d.data_ptr(),
           vocab, lr.data_ptr(), lo.data_ptr(), stream())
    g = torch.full((rows,), -1.0, device="cuda")
    d2 = torch.empty_like(x)
    call_backward(L, x, "f32", t, out["lse"], None, g, None, 1.0, d2)
    # both are p - 1[j = t], p off by 2 E + 4u (|lse| + |ln p|) <= 2 E + 100u in either
    assert float((d - d2).abs().max()) < 2 * (2 * err(vocab, "f32") + 100 * U)
    assert torch.equal(lr, -out["logp"]) or float((lr + out["logp"]).abs().max()) < 2 * err(vocab, "f32") + 100 * U


def test_operators_in_a_graph_and_on_another_stream(L):
    """Captured and replayed on a side stream, each replay of new inputs gives what an eager call gives."""
    rows, vocab, k = 9, 40000, 12
    s = torch.cuda.Stream()
    xs = [make("normal", rows, vocab, "bf16", seed=i) for i in range(3)]
    x = xs[0].clone()
    t = targets_for(rows, vocab)
    ids, v = teacher(rows, vocab, k)
    o = opts(L, scale=0.5)
    lp, en, ls, tl = (torch.empty(n, device="cuda") for n in (rows, rows, rows, rows * k))
    ti = torch.empty(rows * k, device="cuda", dtype=torch.int32)
    gl = torch.ones(rows, device="cuda")
    d1, d2 = torch.empty_like(x), torch.empty_like(x)
    lr, lo = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda")

    def go(st):
        L.call("zl_token_logprobs_bf16", x.data_ptr(), vocab, t.data_ptr(), rows, vocab, 1.0, k, lp.data_ptr(), en.data_ptr(),
               ls.data_ptr(), tl.data_ptr(), ti.data_ptr(), st)
        L.call("zl_token_logprobs_backward_bf16", x.data_ptr(), vocab, t.data_ptr(), ls.data_ptr(), en.data_ptr(), gl.data_ptr(),
               gl.data_ptr(), rows, vocab, 1.0, d1.data_ptr(), vocab, st)
        L.call("zl_distill_topk_bf16", x.data_ptr(), vocab, ids.data_ptr(), v.data_ptr(), k, t.data_ptr(), None, C.byref(o), rows,
               vocab, d2.data_ptr(), vocab, lr.data_ptr(), lo.data_ptr(), st)

    outs = (lp, en, ls, tl, ti, d1, d2, lr, lo)
    want = []
    for z in xs:
        x.copy_(z)
        go(stream())
        want.append([a.clone() for a in outs])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        go(torch.cuda.current_stream().cuda_stream)
    for z, w in zip(xs, want):
        x.copy_(z)
        for a in outs:
            a.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, w):
            assert torch.equal(a, b)


def test_two_streams_at_once(L):
    """Two calls in flight on two streams share nothing."""
    rows, vocab, k = 64, 30000, 20
    xs = [make("normal", rows, vocab, "bf16", seed=i) for i in range(2)]
    t = targets_for(rows, vocab)
    alone = [call_logprobs(L, x, "bf16", t, 1.0, k) for x in xs]
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        both = [call_logprobs(L, x, "bf16", t, 1.0, k, s.cuda_stream) for x, s in zip(xs, ss)]
        torch.cuda.synchronize()
        for (o, a, i), (p, b, j) in zip(alone, both):
            assert torch.equal(a, b) and torch.equal(i, j) and all(torch.equal(o[n], p[n]) for n in o)


def test_zero_rows(L):
    o = opts(L)
    lo = torch.full((1,), 7.0, device="cuda")
    for t in ("bf16", "f32"):
        L.call(f"zl_token_logprobs_{t}", None, 64, None, 0, 64, 1.0, 4, None, None, None, None, lo.data_ptr(), stream())
        L.call(f"zl_token_logprobs_backward_{t}", None, 64, None, None, None, None, None, 0, 64, 1.0, None, 64, stream())
        L.call(f"zl_distill_topk_{t}", None, 64, None, None, 4, lo.data_ptr(), None, C.byref(o), 0, 64, None, 0, None,
               lo.data_ptr(), stream())
        assert float(lo) == 0.0


# ------------------------------------------------------------------ from hidden states
def call_head(L, h, w, t, scale, st=None):
    rows, dim = h.shape
    vocab = w.shape[0]
    out = {n: torch.full((rows + 3,), 7.0, device="cuda") for n in ("logp", "entropy", "lse")}
    ws = torch.empty(max(1, L.load().zl_linear_logprobs_workspace_floats(rows, dim, vocab)), device="cuda")
    L.call("zl_linear_logprobs_bf16", h.data_ptr(), w.data_ptr(), ptr(t), rows, dim, vocab, scale,
           out["logp"].data_ptr() if t is not None else None, out["entropy"].data_ptr(), out["lse"].data_ptr(), ws.data_ptr(),
           st if st is not None else stream())
    torch.cuda.synchronize()
    for v in out.values():
        assert bool((v[rows:] == 7.0).all()), "wrote past its rows"
    return {n: v[:rows] for n, v in out.items()}


def check_head(L, h, w, scale=1.0, t=None):
    """Beside the bounds above a logit is off by at most 2 (dim / 16 + 4) u sum |h w|: products are exact in fp32, and
    each step of 16 adds one rounding (no better than truncation) of a partial sum.  lse and every ln p move by no
    more than the row's largest such error, the entropy by that times (1 + ln vocab + its spread)."""
    rows, dim = h.shape
    vocab = w.shape[0]
    scale = C.c_float(scale).value
    t = targets_for(rows, vocab) if t is None else t
    out = call_head(L, h, w, t, scale)
    x = h.double() @ w.double().T
    logp, lse = softmax64(x, scale)
    off = scale * 2 * (dim / 16 + 4) * U * (h.double().abs() @ w.double().abs().T).amax(1)
    # a thread's sums: chunks of 32 (8 additions to a chain), at most vocab / 64 chunks; 148 partials joined
    E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
    ymax = (x * scale).amax(1)
    close(out["lse"], lse, off + E + 4 * U * (lnv + ymax.abs()), "lse")
    spread = ((logp.exp() * (logp - (logp.exp() * logp).sum(1, keepdim=True)) ** 2).sum(1)).sqrt()
    close(out["entropy"], entropy64(logp), 2 * off * (1 + spread) + E * (2 + lnv) + 4 * U * (lnv + 1), "entropy")
    ok = (t >= 0) & (t < vocab)
    at = logp.gather(1, t.clamp(0, vocab - 1).long()[:, None])[:, 0]
    close(out["logp"], torch.where(ok, at, torch.zeros_like(at)), 2 * off + E + 4 * U * (lnv + at.abs()), "logp")


@pytest.mark.parametrize("rows,dim,vocab", [(1, 8, 1), (1, 64, 2), (2, 512, 6400), (7, 72, 300), (8, 2048, 32000), (9, 520, 1000),
                                            (33, 200, 257), (128, 128, 640), (129, 512, 255), (256, 64, 256), (257, 576, 513),
                                            (300, 1032, 1025), (1000, 512, 6400), (5000, 64, 130), (40, 264, 20011), (1, 1000, 100003),
                                            (300, 512, 45001), (600, 2048, 12000), (2000, 504, 3001),
                                            (8, 8, 15), (5, 24, 17), (3, 8192, 333), (8, 8200, 100), (6, 1048, 50007)])
def test_linear_logprobs_sizes(L, rows, dim, vocab):
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    h = torch.randn(rows, dim, device="cuda", generator=g).bfloat16()
    w = (torch.randn(vocab, dim, device="cuda", generator=g) * (2.5 / math.sqrt(dim))).bfloat16()
    check_head(L, h, w)
    check_head(L, h, w, 0.6)


@pytest.mark.parametrize("rows", [3, 300])
def test_linear_logprobs_values(L, rows):
    """Large logits (every row nearly certain), equal logits, and targets at the edges of the tiles."""
    dim, vocab = 136, 1500
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn(rows, dim, device="cuda", generator=g).bfloat16()
    w = torch.randn(vocab, dim, device="cuda", generator=g).bfloat16()
    edges = torch.tensor([0, 31, 32, 127, 128, 255, 256, 1499, 1500, -5, 1023, 1024], device="cuda", dtype=torch.int32)
    t = edges.repeat(rows // 12 + 1)[:rows].contiguous()
    check_head(L, h * 4, w, t=t)
    check_head(L, h * 0, w, t=t)
    check_head(L, h, w[:1].repeat(vocab, 1).contiguous(), t=t)


def test_linear_logprobs_agrees_with_the_stored_logits(L):
    """On the fp32 logits that the GEMM stores from the same operands, the first operator gives the same."""
    rows, dim, vocab = 70, 512, 6400
    g = torch.Generator(device="cuda").manual_seed(8)
    h = torch.randn(rows, dim, device="cuda", generator=g).bfloat16()
    w = (torch.randn(vocab, dim, device="cuda", generator=g) * 0.1).bfloat16()
    x = torch.empty(rows, vocab, device="cuda")
    e = L.Epilogue()
    L.call("zl_gemm_bf16", h.data_ptr(), w.data_ptr(), x.data_ptr(), rows, vocab, dim, L.A_KMAJOR | L.B_KMAJOR, L.EPI_OUT_F32,
           C.byref(e), None, stream())
    t = targets_for(rows, vocab)
    a, _, _ = call_logprobs(L, x, "f32", t, 1.0, 0)
    b = call_head(L, h, w, t, 1.0)
    off = 4 * (dim / 16 + 4) * U * float((h.double().abs() @ w.double().abs().T).amax())
    for n in a:
        assert float((a[n] - b[n]).abs().max()) < 12 * (off + err(vocab, "f32") + 40 * U)


def test_linear_logprobs_graph_replay(L):
    rows, dim, vocab = 200, 256, 5000
    g = torch.Generator(device="cuda").manual_seed(3)
    hs = [torch.randn(rows, dim, device="cuda", generator=g).bfloat16() for _ in range(2)]
    w = (torch.randn(vocab, dim, device="cuda", generator=g) * 0.1).bfloat16()
    t = targets_for(rows, vocab)
    want = [call_head(L, h, w, t, 1.0) for h in hs]
    h = hs[0].clone()
    out = {n: torch.zeros(rows, device="cuda") for n in ("logp", "entropy", "lse")}
    ws = torch.empty(L.load().zl_linear_logprobs_workspace_floats(rows, dim, vocab), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.call("zl_linear_logprobs_bf16", h.data_ptr(), w.data_ptr(), t.data_ptr(), rows, dim, vocab, 1.0, out["logp"].data_ptr(),
               out["entropy"].data_ptr(), out["lse"].data_ptr(), ws.data_ptr(), stream())
    for z, a in zip(hs, want):
        h.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[n], a[n]) for n in out)


def test_first_calls_inside_a_capture():
    """In a fresh process the first call of every operator may be one that is captured: nothing that an entry sets up
    on its first call is forbidden then."""
    code = """
import ctypes as C, torch
from zerollm_b200 import lib as L
torch.cuda.set_device(0)
V, k, dim, n = 6400, 8, 512, 300
x = torch.randn(n, V, device='cuda').bfloat16()
h = torch.randn(n, dim, device='cuda').bfloat16()
w = (torch.randn(V, dim, device='cuda') * 0.1).bfloat16()
t = torch.randint(0, V, (n,), device='cuda', dtype=torch.int32)
f = [torch.zeros(n, device='cuda') for _ in range(6)]
top, ids = torch.zeros(n, k, device='cuda'), torch.zeros(n, k, device='cuda', dtype=torch.int32)
d, lo = torch.zeros_like(x), torch.zeros(1, device='cuda')
o = L.DistillOptions(0.5, 1.0, 1, 1.0, 0.5, 1.0 / n)
ws = [torch.empty(L.load().zl_linear_logprobs_workspace_floats(r, dim, V), device='cuda') for r in (n, 4)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    p = lambda a: a.data_ptr()
    L.call('zl_token_logprobs_bf16', p(x), V, p(t), n, V, 1.0, k, p(f[0]), p(f[1]), p(f[2]), p(top), p(ids), s)
    L.call('zl_token_logprobs_backward_bf16', p(x), V, p(t), p(f[2]), p(f[1]), p(f[0]), None, n, V, 1.0, p(d), V, s)
    L.call('zl_distill_topk_bf16', p(x), V, p(ids), p(top), k, p(t), None, C.byref(o), n, V, p(d), V, p(f[3]), p(lo), s)
    L.call('zl_linear_logprobs_bf16', p(h), p(w), p(t), n, dim, V, 1.0, p(f[3]), p(f[4]), p(f[5]), p(ws[0]), s)
    L.call('zl_linear_logprobs_bf16', p(h), p(w), p(t), 4, dim, V, 1.0, p(f[3]), p(f[4]), p(f[5]), p(ws[1]), s)
g.replay()
torch.cuda.synchronize()
y = x.float()
assert float((f[2] - torch.logsumexp(y, 1)).abs().max()) < 1e-4
assert float((f[5] - torch.logsumexp(h.float() @ w.float().t(), 1)).abs().max()) < 1e-3
print('captured')
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_short_rows_first_in_a_process():
    """What a kernel is allowed on its first call is not taken as given to another of the same arguments."""
    code = """
import torch
from zerollm_b200 import lib as L
for rows, V, k in ((1500, 300, 64), (4000, 7600, 16)):
    x = torch.randn(rows, V, device='cuda')
    lse, ids = torch.zeros(rows, device='cuda'), torch.zeros(rows, k, device='cuda', dtype=torch.int32)
    L.call('zl_token_logprobs_f32', x.data_ptr(), V, None, rows, V, 1.0, k, None, None, lse.data_ptr(), None, ids.data_ptr(), None)
    torch.cuda.synchronize()
    assert float((lse - torch.logsumexp(x, 1)).abs().max()) < 1e-4
    assert torch.equal(ids.long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k])
print('both')
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "both" in r.stdout, r.stderr[-2000:]


def test_offsets_past_32_bits(L):
    """Rows more than 2^31 elements apart, and a weight of more than 2^31 elements."""
    stride = (1 << 31) // 2 + 1000007
    rows, vocab, k = 4, 3000, 6
    buf = torch.empty(3 * stride + vocab, device="cuda", dtype=torch.bfloat16)
    x = torch.as_strided(buf, (rows, vocab), (stride, 1))
    small = make("normal", rows, vocab, "bf16")
    x.copy_(small)
    t = targets_for(rows, vocab)
    a, at, ai = call_logprobs(L, x, "bf16", t, 1.0, k)
    logp, lse = softmax64(small, 1.0)
    order = torch.sort(small.float(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ai.long(), order)
    close(a["lse"], lse, err(vocab, "bf16") + 4 * U * (math.log(vocab) + lse.abs()), "lse")
    ids, v = teacher(rows, vocab, k)
    o = opts(L)
    lr, lo = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda")
    want, got = torch.empty_like(small), torch.empty_like(small)
    L.call("zl_distill_topk_bf16", small.data_ptr(), vocab, ids.data_ptr(), v.data_ptr(), k, t.data_ptr(), None, C.byref(o), rows,
           vocab, want.data_ptr(), vocab, lr.data_ptr(), lo.data_ptr(), stream())
    L.call("zl_distill_topk_bf16", x.data_ptr(), stride, ids.data_ptr(), v.data_ptr(), k, t.data_ptr(), None, C.byref(o), rows,
           vocab, x.data_ptr(), stride, lr.data_ptr(), lo.data_ptr(), stream())
    got.copy_(x)
    # (the rows lie at other places within 16 bytes: sums in another order, an entry off by a rounding of bf16 at most)
    assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -7 * float(want.double().abs().max())
    x.copy_(small)
    g = torch.ones(rows, device="cuda")
    call_backward(L, x, "bf16", t, a["lse"], None, g, None, 1.0, x)
    call_backward(L, small, "bf16", t, a["lse"], None, g, None, 1.0, want)
    got.copy_(x)
    assert torch.equal(got, want)
    del buf, x
    dim, big = 8192, 270000
    w = torch.empty(big, dim, device="cuda", dtype=torch.bfloat16).normal_(0, 2.0 / math.sqrt(dim))
    for n in (2, 20):
        h = torch.randn(n, dim, device="cuda").bfloat16()
        tt = torch.full((n,), big - 1, device="cuda", dtype=torch.int32)
        out = call_head(L, h, w, tt, 1.0)
        y = torch.cat([h.double() @ c.double().T for c in w.split(30000)], 1)
        lp, ls = softmax64(y, 1.0)
        off = 2 * (dim / 16 + 4) * U * float(h.double().abs().sum(1).max()) * float(w.abs().max())
        assert float((out["lse"] - ls).abs().max()) < off + 1e-3 and float((out["logp"] - lp[:, -1]).abs().max()) < 2 * off + 1e-3


def test_linear_logprobs_on_two_streams(L):
    """Two calls in flight, each with its own workspace, share nothing."""
    g = torch.Generator(device="cuda").manual_seed(6)
    w = (torch.randn(9000, 256, device="cuda", generator=g) * 0.1).bfloat16()
    for rows in (4, 700):
        hs = [torch.randn(rows, 256, device="cuda", generator=g).bfloat16() for _ in range(2)]
        t = targets_for(rows, 9000)
        want = [call_head(L, h, w, t, 1.0) for h in hs]
        n = L.load().zl_linear_logprobs_workspace_floats(rows, 256, 9000)
        ss = [torch.cuda.Stream(), torch.cuda.Stream()]
        ws = [torch.empty(n, device="cuda") for _ in ss]
        outs = [{k: torch.zeros(rows, device="cuda") for k in ("logp", "entropy", "lse")} for _ in ss]
        torch.cuda.synchronize()
        for _ in range(3):
            for h, s, q, o in zip(hs, ss, ws, outs):
                L.call("zl_linear_logprobs_bf16", h.data_ptr(), w.data_ptr(), t.data_ptr(), rows, 256, 9000, 1.0, o["logp"].data_ptr(),
                       o["entropy"].data_ptr(), o["lse"].data_ptr(), q.data_ptr(), s.cuda_stream)
            torch.cuda.synchronize()
            for o, a in zip(outs, want):
                assert all(torch.equal(o[k], a[k]) for k in o)
