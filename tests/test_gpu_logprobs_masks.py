"""Rows masked with finite values, alone and beside -inf, in the operators on next-token distributions: against the
fp64 formulas and with the tolerances of tests/test_gpu_logprobs.py."""
import ctypes as C
import math

import pytest
import torch

from tests.test_gpu_logprobs import (DT, FLUSH, L, NINF, U, call_backward, call_head, call_logprobs,  # noqa: F401
                                     check_distill, check_logprobs, close, entropy64, err, half_step, opts, softmax64, stream,
                                     strided, targets_for)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ alternatives
def mixed_masks(rows, vocab, dtype, ordinary, low, lead, seed=0):
    """Rows of `ordinary` logits and `low` ones of the type's lowest value at random places from `lead` on, the others
    -inf; 1,100 elements of 7, above nearly all of them, lie between the rows and behind the last one."""
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows + vocab)
    x, _ = strided(rows, vocab, dtype, 1100)
    place = torch.rand(rows, vocab - lead, device="cuda", generator=g).argsort(1) + lead
    v = torch.full((rows, vocab), NINF, device="cuda")
    v.scatter_(1, place[:, ordinary:ordinary + low], torch.finfo(DT[dtype]).min)
    v.scatter_(1, place[:, :ordinary], torch.randn(rows, ordinary, device="cuda", generator=g) * 3)
    x.copy_(v)
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(3, 300), (1300, 400), (2400, 1000), (5, 4000), (1300, 4001), (300, 9000), (2, 140000)])
@pytest.mark.parametrize("ordinary,low,lead,k", [(10, 60, 0, 30), (20, 40, 0, 30), (1, 100, 0, 96), (40, 130, 60, 64),
                                                 (0, 200, 0, 25), (24, 24, 200, 48), (120, 1, 0, 128)])
def test_alternatives_beside_lowest_values(L, rows, vocab, ordinary, low, lead, k, dtype):
    """Fewer ordinary logits than alternatives: the others are masks of the lowest value, then -inf, by their index; none
    comes from outside the row."""
    check_logprobs(L, mixed_masks(rows, vocab, dtype, ordinary, low, lead), dtype, 1.0, k, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 1300])
def test_alternatives_behind_a_long_masked_run(L, rows, dtype):
    """Masks of the lowest value in more vectors than are listed at once, behind a run of -inf."""
    for vocab, low, lead in [(3700, 2000, 1700), (8000, 6000, 1600), (30000, 20000, 9000)]:
        check_logprobs(L, mixed_masks(rows, vocab, dtype, 7, low, lead), dtype, 1.0, 40, targets_for(rows, vocab))


# ------------------------------------------------------------------ statistics
MASKS = [-1e4, -1e6, -1e9, -1e10, -1e12, -1e20, -1e30]


def finite_masks(rows, vocab, dtype, value, layout, seed=0):
    """Ordinary logits masked with `value`; the middle row wholly."""
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + vocab)
    x, _ = strided(rows, vocab, dtype)
    v = torch.randn(rows, vocab, device="cuda", generator=g) * 3
    left = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    if layout == "some":
        left |= torch.rand(vocab, device="cuda", generator=g) < 0.6
    elif layout == "few":
        left[torch.randperm(vocab, device="cuda", generator=g)[:5]] = True
    else:                                                     # "behind": whole pieces of masks before the first logit
        left[vocab * 7 // 8:] = True
    left[vocab - 1] = True
    v.masked_fill_(~left, value)
    v[rows // 2] = value
    x.copy_(v)
    return x, left.nonzero()[:, 0]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["some", "few", "behind"])
@pytest.mark.parametrize("value", MASKS)
def test_token_logprobs_finite_masks(L, value, layout, dtype):
    for rows, vocab, k in [(3, 900, 9), (3, 6400, 16), (1300, 1001, 40), (1201, 6400, 0), (600, 9000, 7), (1, 33333, 50),
                           (3, 140000, 64)]:
        x, _ = finite_masks(rows, vocab, dtype, value, layout)
        for scale in (1.0, 0.7):
            check_logprobs(L, x, dtype, scale, k, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", [-1e9, -1e7, -1e5, 1e4, 1e5, 1e6, 1e7, 1e8, 1e9])
def test_token_logprobs_far_from_zero(L, offset, dtype):
    """Rows of ordinary spread about a far value (as far as the type still tells its neighbours apart)."""
    for rows, vocab in [(3, 900), (1300, 640), (2, 50001)]:
        g = torch.Generator(device="cuda").manual_seed(vocab)
        x, _ = strided(rows, vocab, dtype)
        x.copy_(torch.randn(rows, vocab, device="cuda", generator=g, dtype=torch.float64) * 3 + offset)
        for scale in (1.0, 1.3):
            check_logprobs(L, x, dtype, scale, 5, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale,size", [(1e4, 30.0), (1e4, 3000.0), (1e4, 1e-3), (1e3, 10.0), (300.0, 60.0), (1e-4, 3e4), (1e-4, 1e9)])
def test_token_logprobs_extreme_scales(L, scale, size, dtype):
    for rows, vocab in [(3, 900), (1300, 640), (2, 50001)]:
        g = torch.Generator(device="cuda").manual_seed(vocab + 1)
        x, _ = strided(rows, vocab, dtype)
        x.copy_(torch.randn(rows, vocab, device="cuda", generator=g) * size)
        check_logprobs(L, x, dtype, scale, 5, targets_for(rows, vocab))


@pytest.mark.parametrize("rows,dim", [(5, 264), (8, 4096), (9, 264), (300, 520), (40, 2048), (300, 4096), (20, 8200)])
@pytest.mark.parametrize("value", [0.0, 1e4, 1e6, 1e9, 1e20])
def test_linear_logprobs_of_exact_logits(L, rows, dim, value):
    """One entry of hidden is not 0, so a logit is a single product, exact in fp32: tolerances without a product's, the
    same for any number of rows."""
    check_exact_head(L, rows, dim, 5003, value)


@pytest.mark.parametrize("rows,dim,vocab", [(9, 1032, 777), (300, 2048, 1500), (40, 4096, 1001), (260, 8200, 515), (3, 8200, 300),
                                            (300, 520, 700), (20, 768, 1000), (300, 776, 1001), (40, 1536, 600), (40, 1544, 600),
                                            (600, 3000, 2000)])
def test_linear_logprobs_of_long_reductions(L, rows, dim, vocab):
    """Sums of at most 48 steps of 16 (each cut: 2u of its partial sum), joined by one rounding each: a logit is off by at
    most (96 + chunks) u sum |h w|, lse and ln p by the row's largest such error, twice."""
    g = torch.Generator(device="cuda").manual_seed(dim + vocab)
    h = torch.randn(rows, dim, device="cuda", generator=g).bfloat16()
    w = (torch.randn(vocab, dim, device="cuda", generator=g) * (2.5 / math.sqrt(dim))).bfloat16()
    t = targets_for(rows, vocab)
    for a, b in [(h, w), (h.abs(), (w.abs() / 16).bfloat16())]:   # signs at random, and all alike
        out = call_head(L, a, b, t, 1.0)
        x = a.double() @ b.double().T
        logp, lse = softmax64(x, 1.0)
        off = (96 + math.ceil(dim / 64 / 12)) * U * (a.double().abs() @ b.double().abs().T).amax(1)
        E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
        close(out["lse"], lse, off + E + 4 * U * (lnv + x.amax(1).abs()), "lse")
        ok = (t >= 0) & (t < vocab)
        at = logp.gather(1, t.clamp(0, vocab - 1).long()[:, None])[:, 0]
        close(out["logp"], torch.where(ok, at, torch.zeros_like(at)), 2 * off + E + 4 * U * (lnv + at.abs()), "logp")


def exact_head(rows, dim, vocab, value, seed=0):
    """hidden of one entry 1 a row, and a weight of ordinary entries, a third of them -value; column 0 of it is -value
    but for eight entries, so rows with that entry are nearly wholly masked."""
    g = torch.Generator(device="cuda").manual_seed(seed + rows + dim)
    at = torch.randint(0, dim, (rows,), device="cuda", generator=g)
    at[0] = 0
    h = torch.zeros(rows, dim, device="cuda").scatter_(1, at[:, None], 1.0).bfloat16()
    w = torch.randn(vocab, dim, device="cuda", generator=g) * 3
    w = torch.where(torch.rand(vocab, dim, device="cuda", generator=g) < 0.33, torch.full((), -value, device="cuda"), w)
    w[8:, 0] = -value
    w[:, 1] = -value
    if rows > 1:
        h[1] = 0
        h[1, 1] = 1                                           # (wholly masked)
    return h, w.bfloat16()


def check_exact_head(L, rows, dim, vocab, value):
    h, w = exact_head(rows, dim, vocab, value)
    t = targets_for(rows, vocab)
    for scale in (1.0, C.c_float(0.7).value):
        out = call_head(L, h, w, t, scale)
        x = h.double() @ w.double().T
        logp, lse = softmax64(x, scale)
        # a thread's sums: chunks of 32 (8 additions to a chain), at most vocab / 64 chunks; 148 partials joined; terms
        # below the maximum as in the other operators
        E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
        close(out["lse"], lse, E + 4 * U * (lnv + (x * scale).amax(1).abs()), "lse")
        close(out["entropy"], entropy64(logp), E * (2 + lnv) + 4 * U * (lnv + 1), "entropy")
        ok = (t >= 0) & (t < vocab)
        at = logp.gather(1, t.clamp(0, vocab - 1).long()[:, None])[:, 0]
        close(out["logp"], torch.where(ok, at, torch.zeros_like(at)), E + 4 * U * (lnv + at.abs()), "logp")


# ------------------------------------------------------------------ distillation
OPTIONS = [dict(), dict(scale=0.5), dict(scale=0.25), dict(scale=0.7), dict(scale=1.3, ce=0.0)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["some", "few", "behind"])
@pytest.mark.parametrize("value", MASKS)
def test_distill_finite_masks(L, value, layout, dtype):
    for i, (rows, vocab) in enumerate([(5, 900), (5, 6400), (200, 3001), (5, 40001), (3, 140000)]):
        for o in (OPTIONS[i % 5], OPTIONS[(i + 2) % 5]):
            x, left = finite_masks(rows, vocab, dtype, value, layout)
            check_distill(L, x, dtype, min(12, left.numel()), opts(L, **o), columns=left)
            x, _ = finite_masks(rows, vocab, dtype, value, layout)
            check_distill(L, x, dtype, 12, opts(L, **o))          # alternatives the student has masked


def test_distill_finite_masks_of_many_rows(L):
    """More rows than run at once, so that a team's next row follows a wholly masked one."""
    for value in (-1e4, -1e10):
        x, left = finite_masks(4000, 1001, "bf16", value, "behind")
        x[::3] = value
        check_distill(L, x, "bf16", 8, opts(L, scale=0.5), columns=left)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", [-1e9, -1e7, -1e5, 1e4, 1e5, 1e6, 1e7, 1e8, 1e9])
def test_distill_far_from_zero(L, offset, dtype):
    for o in OPTIONS:
        for rows, vocab, dpad in [(5, 901, 0), (3, 50001, 3)]:
            g = torch.Generator(device="cuda").manual_seed(vocab)
            x, _ = strided(rows, vocab, dtype)
            x.copy_(torch.randn(rows, vocab, device="cuda", generator=g, dtype=torch.float64) * 3 + offset)
            check_distill(L, x, dtype, 5, opts(L, **o), dpad=dpad)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale,size", [(1e4, 30.0), (1e4, 1e-3), (1e3, 10.0), (300.0, 60.0), (1e-4, 3e4), (1e-4, 1e9)])
def test_distill_extreme_scales(L, scale, size, dtype):
    for rows, vocab in [(5, 901), (2, 50001)]:
        g = torch.Generator(device="cuda").manual_seed(vocab + 1)
        x, _ = strided(rows, vocab, dtype)
        x.copy_(torch.randn(rows, vocab, device="cuda", generator=g) * size)
        check_distill(L, x, dtype, 5, opts(L, scale=scale))


# ------------------------------------------------------------------ gradient
def check_backward(L, x, dtype, scale, which, dpad=0):
    """Against the fp64 formula on the logits themselves (not on the saved lse, which may round away all of ln vocab):
    p is off by E + (4 + 4 |ln p|) u, its factors by a few u, as in the forward."""
    rows, vocab = x.shape
    scale = C.c_float(scale).value
    t = targets_for(rows, vocab)
    out, _, _ = call_logprobs(L, x, dtype, t, scale, 0)
    g = torch.Generator(device="cuda").manual_seed(4)
    gl = torch.randn(rows, device="cuda", generator=g) if which != "entropy" else None
    ge = torch.randn(rows, device="cuda", generator=g) if which != "logp" else None
    ent = out["entropy"] if ge is not None else None
    d, buf = strided(rows, vocab, dtype, dpad)
    call_backward(L, x, dtype, t, out["lse"], ent, gl, ge, scale, d)
    logp, _ = softmax64(x, scale)
    p = logp.exp()
    l0 = torch.where(p > 0, logp, torch.zeros_like(p))
    ok = (t >= 0) & (t < vocab)
    hot = torch.zeros_like(p).scatter_(1, t.clamp(0, vocab - 1).long()[:, None], 1.0) * ok[:, None]
    gg = (torch.zeros(rows, device="cuda") if gl is None else gl).double() * ok
    h = (torch.zeros(rows, device="cuda") if ge is None else ge).double()
    H = (torch.zeros(rows, device="cuda") if ent is None else ent).double()
    want = scale * (gg[:, None] * (hot - p) - h[:, None] * p * (l0 + H[:, None]))
    size = scale * (gg.abs()[:, None] * (hot + p) + h.abs()[:, None] * p * (l0.abs() + H.abs()[:, None] + 1))
    tol = size * (err(vocab, dtype) + (4 * l0.abs() + 20) * U) + FLUSH * scale * (gg.abs() + h.abs() * (88 + H))[:, None]
    # below kFarLse the saved lse counts, half a step of it
    tol = tol + size * torch.where(out["lse"].abs() <= 256, 2 * U * out["lse"].abs(), torch.zeros_like(out["lse"])).double()[:, None]
    close(d, want, tol + half_step(dtype) * (want.abs() + tol) + FLUSH, "d_logits")
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, d.shape, d.stride(), 0).fill_(False)
    assert bool((buf[mask] == 7.0).all()), "wrote outside its rows"
    y = x.clone() if x.is_contiguous() else x
    call_backward(L, y, dtype, t, out["lse"], ent, gl, ge, scale, y)   # in the logits' place
    if dpad == 0 and x.is_contiguous() and x.data_ptr() % 16 == y.data_ptr() % 16:
        assert torch.equal(y, d)
    else:  # (at another place within 16 bytes: the same formula, sums in another order)
        close(y, want, tol + half_step(dtype) * (want.abs() + tol) + FLUSH, "d_logits in place")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("which", ["logp", "entropy", "both"])
@pytest.mark.parametrize("value", MASKS)
def test_token_logprobs_backward_finite_masks(L, value, which, dtype):
    for rows, vocab, dpad in [(3, 900, 0), (3, 6400, 0), (1300, 1001, 0), (5, 6401, 3), (3, 40001, 0)]:
        x, _ = finite_masks(rows, vocab, dtype, value, "some")
        check_backward(L, x, dtype, 0.7, which, dpad)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset,scale", [(-1e9, 1.0), (-1e5, 1.3), (-270.0, 1.0), (50.0, 1.0), (242.0, 1.0), (300.0, 1.0), (1e3, 0.7),
                                          (1e6, 1.0), (1e8, 1.0), (0.0, 1e4), (0.0, 100.0)])
def test_token_logprobs_backward_far_from_zero(L, offset, scale, dtype):
    for rows, vocab, pad, at, dpad in [(3, 900, 0, 0, 0), (2000, 640, 0, 0, 0), (2, 50001, 0, 0, 0), (5, 1001, 13, 3, 2), (4, 6, 0, 1, 0)]:
        g = torch.Generator(device="cuda").manual_seed(vocab)
        x, _ = strided(rows, vocab, dtype, pad, at)
        x.copy_(torch.randn(rows, vocab, device="cuda", generator=g, dtype=torch.float64) * 3 + offset)
        check_backward(L, x, dtype, scale, "both", dpad)


# ------------------------------------------------------------------ the longest rows
@pytest.mark.parametrize("dtype,vocab", [("bf16", 5505015), ("f32", 1376251)])
def test_alternatives_of_the_longest_rows(L, dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, _ = strided(2, vocab, dtype, 5, 1)
    x.copy_(torch.randn(2, vocab, device="cuda", generator=g) * 3)
    check_logprobs(L, x, dtype, 1.0, 128, targets_for(2, vocab))
    y, _ = strided(2, vocab + 1, dtype)
    y.copy_(torch.randn(2, vocab + 1, device="cuda", generator=g) * 3)
    check_logprobs(L, y, dtype, 1.0, 0, targets_for(2, vocab + 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1.0, 0.5, 0.7])
def test_distill_without_weight_reads_no_record(L, scale, dtype):
    """distill_weight 0 beside a record of NaN, infinities and values beyond any probability: the cross-entropy's loss and
    gradient, the same as without a record."""
    rows, vocab, k = 6, 1001, 9
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(DT[dtype])
    t = targets_for(rows, vocab)
    ids = torch.randint(0, vocab, (rows, k), device="cuda", generator=g, dtype=torch.int32)
    for bad in (math.nan, math.inf, 3e38):
        v = torch.full((rows, k), bad, device="cuda")
        for normalize in (0, 1):
            o = opts(L, scale=scale, kd=0.0, ce=0.7, normalize=normalize)
            got = []
            for n in (k, 0):
                lr, lo, d = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)
                L.call(f"zl_distill_topk_{dtype}", x.data_ptr(), vocab, ids.data_ptr(), v.data_ptr(), n, t.data_ptr(), None,
                       C.byref(o), rows, vocab, d.data_ptr(), vocab, lr.data_ptr(), lo.data_ptr(), stream())
                got.append((lr, lo, d))
            for a, b in zip(*got):
                assert torch.isfinite(a.float()).all() and torch.equal(a, b)


# ------------------------------------------------------------------ maxima that rise
def rising(rows, vocab, dtype, offset):
    """Ascending rows of ordinary spread about `offset`: every piece of a row raises the running maximum."""
    g = torch.Generator(device="cuda").manual_seed(vocab + 7)
    x, _ = strided(rows, vocab, dtype)
    v = torch.randn(rows, vocab, device="cuda", generator=g, dtype=torch.float64).sort(dim=1).values
    x.copy_(v + offset)
    return x


OFFSETS = [-3e5, -5e3, 100.0, 1e3, 3e3, 5e3, 2e4, 9e4, 1.7e5, 3e5]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", OFFSETS)
def test_token_logprobs_of_rising_rows(L, offset, dtype):
    for rows, vocab in [(3, 900), (1300, 3001), (3, 20000), (2, 140000)]:
        for scale in (1.0, 0.7):
            check_logprobs(L, rising(rows, vocab, dtype, offset), dtype, scale, 5, targets_for(rows, vocab))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", OFFSETS)
def test_distill_of_rising_rows(L, offset, dtype):
    for rows, vocab in [(5, 901), (400, 3001), (3, 20000), (2, 140000)]:
        for o in OPTIONS:
            check_distill(L, rising(rows, vocab, dtype, offset), dtype, 5, opts(L, **o))


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("offset", [1e3, 3e3, 5e3, 9e4])
def test_linear_logprobs_of_rising_exact_logits(L, offset, rows):
    """Logits of a single product each, ascending over the vocabulary in steps of bf16."""
    dim, vocab = 136, 3000
    h = torch.zeros(rows, dim, device="cuda")
    h[:, 3] = 1.0
    w = torch.zeros(vocab, dim, device="cuda")
    step = 2.0 ** (math.floor(math.log2(offset)) - 7)
    w[:, 3] = offset + step * torch.arange(vocab, device="cuda").div(200, rounding_mode="floor")
    h, w = h.bfloat16(), w.bfloat16()
    t = targets_for(rows, vocab)
    scale = C.c_float(0.3 / step).value                       # (neighbours 0.3 apart)
    out = call_head(L, h, w, t, scale)
    logp, lse = softmax64(h.double() @ w.double().T, scale)
    E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
    close(out["lse"], lse, E + 4 * U * (lnv + scale * offset * 1.2), "lse")
    close(out["entropy"], entropy64(logp), E * (2 + lnv) + 4 * U * (lnv + 1), "entropy")
    ok = (t >= 0) & (t < vocab)
    at = logp.gather(1, t.clamp(0, vocab - 1).long()[:, None])[:, 0]
    close(out["logp"], torch.where(ok, at, torch.zeros_like(at)), E + 4 * U * (lnv + at.abs()), "logp")


@pytest.mark.parametrize("rows,dim,vocab", [(3, 72, 1000), (8, 72, 17), (9, 72, 1000), (300, 136, 700), (20, 1032, 513)])
def test_linear_logprobs_of_infinite_and_nan_logits(L, rows, dim, vocab):
    """A logit of -inf is masked; one of +inf or NaN makes the statistics NaN; as on stored logits."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.zeros(rows, dim, device="cuda").bfloat16()
    h[:, 5] = 1
    h[rows // 2] = 0
    h[rows // 2, 6] = 1                                       # (another row: column 6 stays finite)
    w = (torch.randn(vocab, dim, device="cuda", generator=g) * 3).bfloat16()
    other = w.clone()
    gone = torch.rand(vocab, device="cuda", generator=g) < 0.5
    gone[vocab // 2] = False
    t = targets_for(rows, vocab)
    E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
    for last in (False, True):                                # masks in the last tile, and everywhere
        z = gone if last else gone & (torch.arange(vocab, device="cuda") >= vocab - 9)
        x = torch.where(z, torch.full((), NINF, device="cuda", dtype=torch.float64), w[:, 5].double())[None].repeat(rows, 1)
        x[rows // 2] = w[:, 6].double()
        # (the rows with column 5 alone: 0 times -inf would be NaN)
        v = other.clone()
        v[z, 5] = NINF
        keep = torch.arange(rows, device="cuda") != rows // 2
        out = call_head(L, h, v, t, 1.0)
        logp, lse = softmax64(x, 1.0)
        close(out["lse"][keep], lse[keep], E + 4 * U * (lnv + 20), "lse")
        close(out["entropy"][keep], entropy64(logp)[keep], E * (2 + lnv) + 4 * U * (lnv + 1), "entropy")
        ok = (t >= 0) & (t < vocab)
        at = logp.gather(1, t.clamp(0, vocab - 1).long()[:, None])[:, 0]
        want = torch.where(ok, at, torch.zeros_like(at))
        close(out["logp"][keep], want[keep], E + 4 * U * (lnv + 20), "logp")
    for bad in (math.inf, math.nan):
        v = other.clone()
        v[vocab // 3, 5] = bad
        out = call_head(L, h, v, t, 1.0)
        assert torch.isnan(out["lse"][keep]).all() and torch.isnan(out["entropy"][keep]).all()
    v = other.clone()
    v[:, 5] = NINF
    out = call_head(L, h, v, t, 1.0)                          # nothing left
    assert bool((out["lse"][keep] == NINF).all()) and bool((out["entropy"][keep] == 0).all())


@pytest.mark.parametrize("rows,dim", [(1, 2048), (4, 4096), (8, 8192), (3, 8192)])
def test_linear_logprobs_of_few_rows_is_as_exact_as_fp32(L, rows, dim):
    """Up to eight rows a logit is a sum of joins of four chains of at most four steps of 16 products (dim a multiple of
    256): off by at most (2 * 4 + dim / 256 + 3) u sum |h w|.  A chain's steps, cut toward zero, shrink it by less than u
    each, which moves the entropy by 4 u times the variance of ln p (2.5^2) over itself (above 6): 5 u; its own sums'
    roundings, at random, add a few u."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    vocab = 8000
    worst = 0.0
    for _ in range(6):
        h = torch.randn(rows, dim, device="cuda", generator=g).bfloat16()
        w = (torch.randn(vocab, dim, device="cuda", generator=g) * (2.5 / math.sqrt(dim))).bfloat16()
        t = targets_for(rows, vocab)
        out = call_head(L, h, w, t, 1.0)
        x = h.double() @ w.double().T
        logp, lse = softmax64(x, 1.0)
        off = (8 + dim / 256 + 3) * U * (h.double().abs() @ w.double().abs().T).amax(1)
        E, lnv = (8 + math.ceil(vocab / 64) + 5 * 20) * U, math.log(vocab)
        close(out["lse"], lse, off + E + 4 * U * (lnv + x.amax(1).abs()), "lse")
        worst = max(worst, float((out["entropy"].double() - entropy64(logp)).norm() / entropy64(logp).norm()))
    assert worst < 16 * U
