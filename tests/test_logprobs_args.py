"""Refusals of the operators on next-token distributions, all on the host before any device work (the
pointers here are never dereferenced)."""
import ctypes as C
import math

import pytest

A = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def L():
    from zerollm_b200 import lib
    lib.load()
    return lib


def refused(L, name, code, word, *args):
    st = getattr(L.load(), name)(*args)
    assert st == code, (name, st, L.load().zl_last_error())
    assert word in L.load().zl_last_error().decode()


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_token_logprobs_refusals(L, t):
    n = "zl_token_logprobs_" + t

    def args(x=A, stride=100, tg=A, rows=4, vocab=100, scale=1.0, k=5, logp=A, ids=A):
        return (x, stride, tg, rows, vocab, scale, k, logp, A, A, A, ids, None)

    bad = L.ZL_EINVAL
    refused(L, n, bad, "sizes", *args(rows=-1))
    refused(L, n, bad, "sizes", *args(vocab=0))
    refused(L, n, bad, "stride", *args(stride=99))
    for s in (0.0, -1.0, math.nan, math.inf, 1e-5, 1e5):
        refused(L, n, bad, "scale", *args(scale=s))
    refused(L, n, bad, "null logits", *args(x=None))
    refused(L, n, bad, "element boundary", *args(x=A + 1))
    refused(L, n, bad, "targets", *args(tg=None))
    refused(L, n, bad, "top_k", *args(k=-1))
    refused(L, n, bad, "top_k", *args(k=101))
    refused(L, n, L.ZL_EUNSUPPORTED, "top_k", *args(k=129, vocab=200, stride=200))
    refused(L, n, bad, "top_ids", *args(ids=None))
    refused(L, n, bad, "4-byte", *args(tg=A + 2))
    refused(L, n, bad, "4-byte", *args(ids=A + 1))
    refused(L, n, L.ZL_EUNSUPPORTED, "2^30", *args(vocab=(1 << 30) + 1, stride=1 << 31))
    assert getattr(L.load(), n)(*args(rows=0, x=None)) == L.ZL_OK


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_token_logprobs_backward_refusals(L, t):
    n = "zl_token_logprobs_backward_" + t

    def args(x=A, stride=100, tg=A, lse=A, ent=A, gl=A, ge=A, rows=4, vocab=100, scale=1.0, d=2 * A, ds=100):
        return (x, stride, tg, lse, ent, gl, ge, rows, vocab, scale, d, ds, None)

    bad = L.ZL_EINVAL
    refused(L, n, bad, "sizes", *args(vocab=-3))
    refused(L, n, bad, "stride", *args(stride=50))
    refused(L, n, bad, "stride", *args(ds=50))
    refused(L, n, bad, "scale", *args(scale=0.0))
    refused(L, n, bad, "null", *args(d=None))
    refused(L, n, bad, "null", *args(lse=None))
    refused(L, n, bad, "element boundary", *args(d=A + 1))
    refused(L, n, bad, "targets", *args(tg=None))
    refused(L, n, bad, "entropies", *args(ent=None))
    refused(L, n, bad, "4-byte", *args(gl=A + 2))
    refused(L, n, bad, "row stride", *args(d=A, ds=101))
    assert getattr(L.load(), n)(*args(rows=0, x=None, d=None, lse=None)) == L.ZL_OK


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_distill_refusals(L, t):
    n = "zl_distill_topk_" + t

    def args(x=A, stride=100, ids=A, v=A, k=5, tg=A, opt=(1.0, 1.0, 1, 0.5, 0.5, 1.0), rows=4, vocab=100, d=2 * A, ds=100,
             lr=A, lo=A):
        o = L.DistillOptions(*opt) if opt else None
        return (x, stride, ids, v, k, tg, None, C.byref(o) if o else None, rows, vocab, d, ds, lr, lo, None)

    bad = L.ZL_EINVAL
    refused(L, n, bad, "options", *args(opt=None))
    refused(L, n, bad, "sizes", *args(rows=-2))
    refused(L, n, bad, "stride", *args(stride=99))
    refused(L, n, bad, "stride", *args(ds=99))
    refused(L, n, bad, "scale", *args(opt=(0.0, 1.0, 1, 0.5, 0.5, 1.0)))
    refused(L, n, bad, "teacher_scale", *args(opt=(1.0, math.nan, 1, 0.5, 0.5, 1.0)))
    for i in (3, 4, 5):
        o = [1.0, 1.0, 1, 0.5, 0.5, 1.0]
        o[i] = math.inf
        refused(L, n, bad, "finite", *args(opt=o))
    refused(L, n, bad, "top_k", *args(k=-1))
    refused(L, n, L.ZL_EUNSUPPORTED, "top_k", *args(k=129))
    refused(L, n, bad, "teacher", *args(ids=None))
    refused(L, n, bad, "teacher", *args(v=None))
    refused(L, n, bad, "targets", *args(tg=None))
    refused(L, n, bad, "element boundary", *args(d=A + 1))
    refused(L, n, bad, "row stride", *args(d=A, ds=104))
    refused(L, n, bad, "loss_rows", *args(lr=None))
    refused(L, n, bad, "4-byte", *args(ids=A + 2))
    refused(L, n, bad, "4-byte", *args(lo=A + 3))


def test_linear_logprobs_refusals(L):
    n = "zl_linear_logprobs_bf16"

    def args(h=A, w=A, tg=A, rows=4, dim=64, vocab=100, scale=1.0, logp=A, ws=A):
        return (h, w, tg, rows, dim, vocab, scale, logp, A, A, ws, None)

    bad = L.ZL_EINVAL
    refused(L, n, bad, "sizes", *args(rows=-1))
    refused(L, n, bad, "sizes", *args(dim=0))
    refused(L, n, bad, "sizes", *args(vocab=0))
    refused(L, n, L.ZL_EUNSUPPORTED, "dim", *args(dim=60))
    refused(L, n, bad, "scale", *args(scale=math.nan))
    refused(L, n, bad, "targets", *args(tg=None))
    refused(L, n, bad, "null", *args(ws=None))
    refused(L, n, bad, "null", *args(h=None))
    refused(L, n, bad, "aligned", *args(w=A + 8))
    refused(L, n, bad, "aligned", *args(ws=A + 4))
    refused(L, n, bad, "4-byte", *args(tg=A + 1))
    refused(L, n, L.ZL_EUNSUPPORTED, "2^30", *args(vocab=(1 << 30) + 1))
    refused(L, n, L.ZL_EUNSUPPORTED, "2^30", *args(rows=(1 << 31) - 1))
    assert getattr(L.load(), n)(*args(rows=0, h=None, w=None, ws=None)) == L.ZL_OK


def test_linear_logprobs_workspace(L):
    """A partial (four floats, two halves of a tile's columns) of every row for each pair of SMs that can meet its row
    tile: at least one, no more than the vocabulary has tiles of 256 (one more where segments do not begin with the row
    tile).  Up to eight rows: one for each block of 128 vocabulary entries, at most two blocks an SM."""
    f = L.load().zl_linear_logprobs_workspace_floats
    for rows, vocab in [(300, 6400), (32768, 6400), (16384, 32000)]:
        n = f(rows, 512, vocab)
        assert n % (rows * 8) == 0 and 1 <= n // (rows * 8) <= (vocab + 255) // 256 + 1
    for rows, vocab in [(1, 1), (1, 32000), (8, 6400)]:
        n = f(rows, 512, vocab)
        assert n % (rows * 4) == 0 and 1 <= n // (rows * 4) <= (vocab + 127) // 128
    assert f(0, 512, 100) == 0 and f((1 << 31) - 1, 512, 100) == 0


def test_model_entries_refuse_null_arguments(L):
    o = L.DistillOptions(1.0, 1.0, 1, 0.5, 0.5, 1.0)
    refused(L, "zl_model_distill_step", L.ZL_EINVAL, "null", None, A, A, A, 4, A, None, C.byref(o), 1, 128, 0.0, 1, None, None)
    refused(L, "zl_model_score", L.ZL_EINVAL, "null", None, A, A, 1, 128, 1.0, 0, A, A, A, None, None, None)


@pytest.mark.parametrize("t,most", [("bf16", 5505015), ("f32", 1376251)])
def test_alternatives_of_very_long_rows(L, t, most):
    """The longest row whose alternatives are found, and one more: refused before anything runs, with no rows too (as
    a model's scoring asks before its forward)."""
    n = "zl_token_logprobs_" + t
    f = getattr(L.load(), n)
    for rows in (0, 2):
        refused(L, n, L.ZL_EUNSUPPORTED, "alternatives", A, most + 1, A, rows, most + 1, 1.0, 1, A, A, A, A, A, None)
    assert f(A, most, A, 0, most, 1.0, 1, A, A, A, A, A, None) == L.ZL_OK
    assert f(A, most + 1, A, 0, most + 1, 1.0, 0, A, A, A, None, None, None) == L.ZL_OK
