"""The model's paths over the operators on next-token distributions: scoring, the distillation step, the trainer
with a teacher, and the numpy front-end."""
import json
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GRAD_TOL = 2e-2   # the model tests' bar on bf16 gradients


def rel(a, b):
    a, b = np.asarray(a, np.float64).ravel(), np.asarray(b, np.float64).ravel()
    return float(np.max(np.abs(a - b)) / max(np.max(np.abs(b)), 1e-30))


def make(tied=0, seed=3, B=3, S=128, vocab=576):
    from zerollm_b200 import Config, ZeroLLM
    c = Config(vocab_size=vocab, embed_dim=128, num_layers=2, num_heads=2, ff_hidden_dim=256, max_seq_len=S, tied=tied)
    m = ZeroLLM(c, B * S, seed=seed, init_std=0.15)
    m.set_optimizer()
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, (B * S,), device="cuda", generator=g, dtype=torch.int32)
    tg = torch.randint(0, vocab, (B * S,), device="cuda", generator=g, dtype=torch.int32)
    return m, ids, tg


def formulas(logits, tg, scale):
    lp = torch.log_softmax(logits.double() * scale, 1)
    return {"logp": lp.gather(1, tg.long()[:, None])[:, 0], "entropy": -(lp.exp() * lp).sum(1),
            "lse": torch.logsumexp(logits.double() * scale, 1)}, lp


@pytest.mark.parametrize("tied", [0, 1])
@pytest.mark.parametrize("B,S", [(3, 128), (1, 1), (1, 8), (2, 100)])
def test_score_matches_the_logits_of_forward(tied, B, S):
    """Without alternatives the head's fp32 sums are scored, which zl_model_forward stores: both are sums of the same
    bf16 products in another order, off by less than 4 (dim / 16 + 4) u sum |h w| each (as in the operators' tests);
    |h| is about sqrt(dim) after the norm and |w| 0.15 sqrt(dim), so sum |h w| < dim."""
    m, ids, tg = make(tied=tied, B=3, S=128)
    n, V, dim = B * S, 576, 128
    logits = torch.empty(n, V, device="cuda")
    got = m.score(ids, tg, B, S, scale=0.9)
    m.forward(ids, B, S, logits)
    want, _ = formulas(logits, tg[:n], float(np.float32(0.9)))
    off = 2 * 4 * (dim / 16 + 4) * U * dim
    for k in want:
        assert float((got[k].double() - want[k]).abs().max()) < (1 + math.log(V)) * off + 400 * U
    m.close()


def test_score_with_alternatives_uses_the_step_logits():
    """With alternatives the bf16 logits are scored: each off by half a bf16 step (2^-9 |x| of a value's spacing)."""
    m, ids, tg = make()
    n, V, k = 384, 576, 9
    logits = torch.empty(n, V, device="cuda")
    got = m.score(ids, tg, 3, 128, top_k=k)
    m.forward(ids, 3, 128, logits)
    want, lp = formulas(logits, tg, 1.0)
    off = 2.0 ** -8 * float(logits.abs().max())
    for key in want:
        assert float((got[key].double() - want[key]).abs().max()) < 2 * (1 + math.log(V)) * off
    x16 = logits.bfloat16().float()
    order = torch.sort(x16, dim=1, descending=True, stable=True)
    # the fp32 logits of the two products round to the same bf16 but where one lies at a border: nearly all ids agree
    assert float((got["top_ids"].long() == order.indices[:, :k]).float().mean()) > 0.98
    at = lp.gather(1, got["top_ids"].long())
    assert float((got["top_logp"].double() - at).abs().max()) < 2 * (1 + math.log(V)) * off
    m.close()


def test_score_on_a_side_stream_and_between_steps():
    """Scoring changes nothing that a later step computes, and runs on the stream it is given."""
    a, ids, tg = make()
    b, _, _ = make()
    s = torch.cuda.Stream()
    for i in range(3):
        la = float(a.train_step(ids, tg, 3, 128, 1e-3))
        torch.cuda.synchronize()
        got = b.score(ids, tg, 3, 128, stream=s)
        s.synchronize()
        lb = float(b.train_step(ids, tg, 3, 128, 1e-3))
        # the mean of -ln p before the step is the step's loss (bf16 logits there: 2^-8 of their size)
        assert abs(-float(got["logp"].double().mean()) - lb) < 2.0 ** -8 * 40
        assert abs(la - lb) <= 1e-4 * abs(la)   # (the steps' atomics may add in another order)
    a.close()
    b.close()


def test_distill_step_on_hard_targets_is_the_training_step():
    """distill_weight 0 and target_weight 1: the cross-entropy step, with logit gradients equal but for their bf16
    rounding."""
    m, ids, tg = make()
    l0 = float(m.train_step(ids, tg, 3, 128, 0.0, update=False))
    g0 = m.grads()
    t_ids = torch.zeros(384, 4, device="cuda", dtype=torch.int32)
    t_val = torch.zeros(384, 4, device="cuda")
    l1 = float(m.distill_step(ids, t_ids, t_val, tg, 3, 128, 0.0, distill_weight=0.0, target_weight=1.0, update=False))
    g1 = m.grads()
    assert abs(l0 - l1) < 1e-5 * abs(l0)
    assert rel(g1, g0) < GRAD_TOL
    m.close()


def test_distill_step_matches_forward_loss_backward():
    """The step against its pieces: forward to fp32 logits, the fp32 operator, backward of its gradient.  The step's
    logits are bf16, so entries of the gradients differ at the model tests' bf16 bar, the loss by the logits' rounding
    (2^-9 of their size at most, on average)."""
    from zerollm_b200 import lib as L
    import ctypes as C
    m, ids, tg = make()
    teacher, _, _ = make(seed=8)
    n, V, k, s = 384, 576, 12, 0.5
    rec = teacher.score(ids, None, 3, 128, scale=s, top_k=k)
    w = torch.ones(n, device="cuda")
    w[::7] = 0.0
    args = dict(scale=s, distill_weight=3.0, target_weight=0.25, row_weight=w)
    loss = float(m.distill_step(ids, rec["top_ids"], rec["top_logp"], tg, 3, 128, 0.0, update=False, **args))
    g = m.grads()
    logits, d = torch.empty(n, V, device="cuda"), torch.empty(n, V, device="cuda")
    m.zero_grad()
    m.forward(ids, 3, 128, logits)
    lr, lo = torch.empty(n, device="cuda"), torch.empty(1, device="cuda")
    o = L.DistillOptions(s, 1.0, 1, 3.0, 0.25, 1.0 / n)
    L.call("zl_distill_topk_f32", logits.data_ptr(), V, rec["top_ids"].data_ptr(), rec["top_logp"].data_ptr(), k, tg.data_ptr(),
           w.data_ptr(), C.byref(o), n, V, d.data_ptr(), V, lr.data_ptr(), lo.data_ptr(), torch.cuda.current_stream().cuda_stream)
    m.backward(ids, d, 3, 128)
    torch.cuda.synchronize()
    assert abs(loss - float(lo)) < 2.0 ** -9 * float(logits.abs().max()) * 3.25
    assert rel(g, m.grads()) < GRAD_TOL
    # and with an update the weights move
    before = m.params()
    m.distill_step(ids, rec["top_ids"], rec["top_logp"], None, 3, 128, 1e-3, scale=s)
    assert not np.array_equal(before, m.params())
    m.close()
    teacher.close()


def test_model_entries_refuse_before_they_run():
    from zerollm_b200 import ZLError
    m, ids, tg = make()
    t_ids = torch.zeros(384, 4, device="cuda", dtype=torch.int32)
    t_val = torch.zeros(384, 4, device="cuda")
    before = m.grads()
    with pytest.raises(ZLError):
        m.distill_step(ids, t_ids, t_val, None, 3, 128, 0.0, target_weight=1.0)     # a target weight without targets
    with pytest.raises(ZLError):
        m.distill_step(ids, t_ids, t_val, tg, 3, 128, 0.0, scale=0.0)
    with pytest.raises(ZLError):
        m.score(ids, tg, 3, 256)                                                    # beyond the model's context
    with pytest.raises(ZLError):
        m.score(ids, tg, 3, 128, top_k=200)
    assert np.array_equal(before, m.grads())
    m.close()


def test_trainer_with_a_teacher(tmp_path):
    """The trainer's command with --teacher runs its steps, logs finite losses and saves a checkpoint; the steps are
    the model's distillation steps on the teacher's record."""
    from zerollm_b200 import ZeroLLM
    from zerollm_b200.model import Config
    from zerollm_b200 import trainer
    cfg = Config(vocab_size=256, embed_dim=128, num_layers=2, num_heads=2, ff_hidden_dim=256, max_seq_len=128)
    t = ZeroLLM(cfg, 512, seed=11)
    t.save(str(tmp_path / "teacher"))
    tokens, offsets = trainer.synthetic_stories(60, 150, 64, seed=4)
    tr = trainer.Trainer(cfg, tokens, offsets, batch=4, seq=128, lr=1e-3, seed=1, teacher=str(tmp_path / "teacher"),
                         teacher_top_k=8, teacher_weight=0.75, temperature=2.0)
    assert np.array_equal(tr.teacher.params(), t.params())
    logs = []
    assert np.isfinite(tr.epoch(max_steps=2, log_every=1, log=logs.append)) and len(logs) == 2
    assert all(np.isfinite(json.loads(x)["loss"]) for x in logs)
    tr.close()
    t.close()
    big = ZeroLLM(Config.baseline_26m(), 512, seed=2)
    big.save(str(tmp_path / "big"))
    big.close()
    rc = trainer.main(["--synthetic", "40", "--batch", "2", "--seq", "256", "--max-steps", "2", "--log-every", "1", "--teacher",
                       str(tmp_path / "big"), "--temperature", "2", "--save", str(tmp_path / "ck")])
    assert rc == 0 and (tmp_path / "ck" / "config.bin").exists()


def test_numpy_front_end():
    from zerollm_b200 import kernels as K
    rng = np.random.default_rng(0)
    M, N, k = 5, 333, 7
    x = rng.standard_normal((M, N)).astype(np.float32)
    t = np.array([0, 5, 332, -1, 9], np.int32)
    logp, ent, lse, top, ids = K.token_logprobs(x, t, M, N, 0.5, k)
    lp = x.astype(np.float64) * 0.5
    lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
    has = (t >= 0)
    tol = 500 * U * 8
    assert np.abs(logp - np.where(has, lp[np.arange(M), np.clip(t, 0, N - 1)], 0)).max() < tol
    assert np.abs(ent + (np.exp(lp) * lp).sum(1)).max() < tol
    assert np.array_equal(ids, np.argsort(-x, axis=1, kind="stable")[:, :k])
    assert np.abs(top - np.take_along_axis(lp, ids.astype(np.int64), 1)).max() < tol
    assert K.token_logprobs(x, t, M, N)[2].shape == (M,)
    g = rng.standard_normal(M).astype(np.float32)
    d = K.token_logprobs_backward(x, t, lse, ent, g, None, M, N, 0.5).reshape(M, N)
    hot = np.zeros((M, N))
    hot[np.arange(M)[has], t[has]] = 1
    want = 0.5 * (g * has)[:, None] * (hot - np.exp(lp))
    assert np.abs(d - want).max() < tol * np.abs(g).max()
    rows, loss, dx = K.distill_topk(x, ids, top, k, t, M, N, scale=0.5, distill_weight=0.0, target_weight=1.0, grad_scale=0.25)
    l1 = x.astype(np.float64) - np.log(np.exp(x.astype(np.float64)).sum(1, keepdims=True))
    want = np.where(has, -l1[np.arange(M), np.clip(t, 0, N - 1)], 0)
    assert np.abs(rows - want).max() < tol and abs(loss - 0.25 * want.sum()) < tol * M
    assert np.abs(dx.reshape(M, N) - 0.25 * has[:, None] * (np.exp(l1) - hot)).max() < tol


def test_score_on_another_stream_has_memory_of_its_own():
    """The outputs of a call on another stream do not lie in memory that a kernel of the current stream, still under way,
    will write: memory freed there belongs to that stream."""
    m, ids, tg = make()
    want = m.score(ids, tg, 3, 128, top_k=5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    m.score(ids, tg, 3, 128, top_k=5, stream=s)
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)                         # some 10 ms
        old = [torch.full((384,), 7.0, device="cuda") for _ in range(8)] + [torch.full((384, 5), 7.0, device="cuda") for _ in range(4)]
        del old                                               # freed, but written only when the sleep is over
        got = m.score(ids, tg, 3, 128, top_k=5, stream=s)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), k
    m.close()


def test_tensors_of_another_kind_are_refused():
    """Ids as topk() gives them (64 bits), transposed records, other types, counts and devices are no arrays that the
    library may read by their address."""
    m, ids, tg = make()
    n, k = 384, 4
    t_ids = torch.zeros(n, k, device="cuda", dtype=torch.int32)
    t_val = torch.zeros(n, k, device="cuda")
    w = torch.ones(n, device="cuda")
    before = m.grads()
    for args, kw in [((t_ids.long(), t_val, tg), {}), ((t_ids, t_val.bfloat16(), tg), {}), ((t_ids, t_val.T.contiguous().T, tg), {}),
                     ((t_ids[:200], t_val[:200], tg), {}), ((t_ids.cpu(), t_val, tg), {}), ((t_ids, t_val, tg.long()), {}),
                     ((t_ids, t_val, tg[:100]), {}), ((t_ids, t_val, tg), dict(row_weight=w[:5])),
                     ((t_ids, t_val, tg), dict(row_weight=w.double()))]:
        with pytest.raises(AssertionError):
            m.distill_step(ids, *args, 3, 128, 0.0, **kw)
    for bad in (tg.long(), tg[:100], tg.cpu()):
        with pytest.raises(AssertionError):
            m.score(ids, bad, 3, 128)
    assert np.array_equal(before, m.grads())
    m.close()


@pytest.mark.parametrize("T,weight,k", [(2.0, 0.75, 8), (1.0, 0.3, 3), (4.0, 1.0, 20)])
def test_trainer_step_is_the_distillation_step(tmp_path, T, weight, k):
    """A step of the trainer with a teacher: loss and gradients of the explicit calls on a model of the same weights, and
    the loss by its formula from both models' fp32 logits.  The step's logits are bf16: each is off by at most half a step
    of the largest one (2^-8 of its power of two), a student's ln p by twice that at scale 1 / T, a teacher's q by twice
    that of itself, so q (ln q - ln p) by four of them times (1 + |ln q - ln p|)."""
    from zerollm_b200 import Config, ZeroLLM, trainer
    cfg = Config(vocab_size=256, embed_dim=128, num_layers=2, num_heads=2, ff_hidden_dim=256, max_seq_len=128)
    B, S, V = 4, 128, 256
    t = ZeroLLM(cfg, B * S, seed=11, init_std=0.1)
    t.save(str(tmp_path / "teacher"))
    tokens, offsets = trainer.synthetic_stories(60, 150, 64, seed=4)
    tr = trainer.Trainer(cfg, tokens, offsets, batch=B, seq=S, lr=1e-3, seed=1, teacher=str(tmp_path / "teacher"),
                         teacher_top_k=k, teacher_weight=weight, temperature=T)
    m = ZeroLLM(cfg, B * S, seed=5, init_std=0.1)
    m.set_optimizer()
    tr.model.set_params(m.params())
    g = torch.Generator(device="cuda").manual_seed(2)
    tr.d_ids.copy_(torch.randint(0, V, (B * S,), device="cuda", generator=g))
    tr.d_tg.copy_(torch.randint(0, V, (B * S,), device="cuda", generator=g))
    ls, lt = torch.empty(B * S, V, device="cuda"), torch.empty(B * S, V, device="cuda")
    m.forward(tr.d_ids, B, S, ls)
    t.forward(tr.d_ids, B, S, lt)
    rec = t.score(tr.d_ids, None, B, S, 1.0 / T, k)
    at = rec["top_ids"].long()
    lq = torch.log_softmax(lt.double().gather(1, at) / T, 1)
    lp = torch.log_softmax(ls.double() / T, 1).gather(1, at)
    ce = -torch.log_softmax(ls.double(), 1).gather(1, tr.d_tg.long()[:, None]).mean()
    want = weight * T * T * (lq.exp() * (lq - lp)).sum(1).mean() + (1 - weight) * ce
    loss = float(tr.train_step())
    got = tr.model.grads()
    other = float(m.distill_step(tr.d_ids, rec["top_ids"], rec["top_logp"], tr.d_tg, B, S, 1e-3, scale=1.0 / T,
                                 distill_weight=weight * T * T, target_weight=1.0 - weight))
    assert abs(loss - other) <= 1e-5 * abs(other) and rel(got, m.grads()) < GRAD_TOL
    step = 2.0 ** (math.floor(math.log2(float(torch.maximum(ls.abs().amax(), lt.abs().amax())))) - 8)
    slack = weight * T * T * 4 * step / T * (1 + float((lq - lp).abs().max())) + (1 - weight) * 2 * step
    assert abs(loss - float(want)) < slack
    # a step on the cross-entropy alone would fail: its loss is within 2 step of ce, and slack >= step (4 weight T + 2 - 2
    # weight) >= 2 step for T >= 1/2, so it is more than 2 slack - slack from the loss wanted
    assert abs(float(want) - float(ce)) > 2 * slack
    tr.close()
    t.close()
    m.close()
