"""Token scores and distillation as a training loop uses them: a teacher engine's forward pass is scored, its top
alternatives become the target of a student engine, whose backward pass and optimiser then run from the gradient that
the distillation wrote where the plan's own loss would have written it. Against the oracle's forward and backward pass
around a 64-bit distillation."""
import ctypes as C

import numpy as np
import pytest

import tccase
import tol
import token_ref as R
from oracle import pyoracle as O
from see_ml_b200 import _lib as L
from see_ml_b200 import formats as F
from see_ml_b200 import plansynth as PS

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _case():
    lib = L.lib()
    model, spec, toks = tccase.build()
    blob, info = PS.synthesize(model, spec, hasher=lambda b, o: int(
        lib.seeml_b200_plan_self_hash(np.frombuffer(b, np.uint8).ctypes.data, len(b), o)))
    return blob, info, toks


@pytest.mark.parametrize("mode", [1, 0], ids=["fused", "contract"])
def test_teacher_scores_feed_a_student_step(mode):
    from see_ml_b200.engine import UpdateEngine
    lib = L.lib()
    blob, info, toks = _case()
    plan = F.parse_plan(blob)
    h = plan.header
    ops = plan.train["opcode"]
    fwd = int(np.nonzero(ops == int(F.Op.XENT_FWD))[0][0])
    bwd = int(np.nonzero(ops == int(F.Op.XENT_BWD))[0][0])
    opt = int(np.nonzero(ops == int(F.Op.ADAMW))[0][0])
    rows, vocab = (int(v) for v in plan.train["out"][fwd, :2])
    logits_ref, dlogits_ref = int(plan.train["in"][fwd, 0]), int(plan.train["in"][bwd, 3])
    per = h.batch // tccase.S
    recs = toks[:per]
    tok, lab = (np.ascontiguousarray(recs[:, s]).reshape(-1) for s in (slice(None, -1), slice(1, None)))
    K, T = 12, 2.0
    weight = np.ones(rows, np.float32)
    weight[rows - 37:] = 0.0                                   # a padded batch
    weight_d = torch.from_numpy(weight).cuda()
    tid = torch.empty(rows, K, dtype=torch.int32, device="cuda")
    tlp = torch.empty(rows, K, device="cuda")
    row_loss, loss = torch.empty(rows, device="cuda"), torch.empty((), device="cuda")
    logprob, entropy = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    torch.cuda.synchronize()

    def values(seed):
        rng = np.random.default_rng(seed)
        return {ad["b_ref"]: (rng.standard_normal(ad["r"] * ad["m"]) * 0.05).astype(np.float32) for ad in info.adapters}

    def engine(seed):
        e = UpdateEngine(0, mode, 0)
        e.load_from_memory(blob)
        for ref, v in values(seed).items():
            e.arena_write(ref, v)
        e.arena_write(h.input_ref, tok)
        e.arena_write(h.label_ref, lab)
        e.run_train_range(0, fwd)
        base = lib.seeml_b200_ctx_arena(C.c_void_p(e.ctx()))
        return e, base, C.c_void_p(lib.seeml_b200_ctx_stream(C.c_void_p(e.ctx())))

    teacher, base, stream = engine(1)
    d = L.TokenScores(base + logits_ref, base + h.label_ref, logprob.data_ptr(), entropy.data_ptr(), None, tlp.data_ptr(),
                      tid.data_ptr(), rows, vocab, vocab, 0, K, T, 0)
    L.check(lib.seeml_b200_token_scores_fwd(C.byref(d), stream))
    L.check(lib.seeml_b200_sync(C.c_void_p(teacher.ctx())))
    teacher_logits = teacher.arena_read(logits_ref, rows * vocab * 4).view(np.float32).reshape(rows, vocab).astype(np.float64)
    lp, H, top_lp, top_id = R.scores(teacher_logits, lab, K, T)
    np.testing.assert_array_equal(tid.cpu().numpy(), top_id)
    bar = R.delta(vocab)
    assert np.abs(logprob.double().cpu().numpy() - lp).max() <= bar + R.U * np.abs(lp).max()
    assert np.abs(tlp.double().cpu().numpy() - top_lp).max() <= bar + R.U * np.abs(top_lp).max()
    assert np.abs(entropy.double().cpu().numpy() - H).max() <= 2 * (1 + np.log(vocab)) * bar + R.U * H.max()
    teacher.close()

    student, base, stream = engine(2)
    student_logits = student.arena_read(logits_ref, rows * vocab * 4).view(np.float32).reshape(rows, vocab).astype(np.float64)
    scale = 1.0                                                # gradients of unit scale, which the tolerance is stated for
    q = L.DistillTopk(base + logits_ref, tid.data_ptr(), tlp.data_ptr(), weight_d.data_ptr(), row_loss.data_ptr(),
                      loss.data_ptr(), None, base + dlogits_ref, rows, vocab, vocab, vocab, 0, 0, K, 1, T, scale)
    L.check(lib.seeml_b200_distill_topk_fwd(C.byref(q), stream))
    student.run_train_range(bwd + 1, opt)
    L.check(lib.seeml_b200_sync(C.c_void_p(student.ctx())))

    # the oracle's stream around the same step
    want = np.zeros(F.align_up(h.arena_size), np.uint8)
    want[:h.persist_init_size] = plan.persist_init
    for ref, v in values(2).items():
        want[ref:ref + v.nbytes] = v.view(np.uint8)
    want[h.input_ref:h.input_ref + tok.nbytes] = tok.view(np.uint8)
    want[h.label_ref:h.label_ref + lab.nbytes] = lab.view(np.uint8)
    O.execute("port", plan.train[:fwd], want, np.asarray(plan.rodata))
    tol.assert_close(student_logits, want[logits_ref:logits_ref + rows * vocab * 4].view(np.float32), "logits")
    row, err, grad, _ = R.distill(student_logits, tid.cpu().numpy(), tlp.double().cpu().numpy(), T, True)
    total = scale * (row * weight).sum()
    assert abs(loss.item() - total) <= scale * ((err + np.abs(row) * R.U) * weight).sum() + R.U * abs(total)
    dlogits = (grad * (scale * weight)[:, None]).astype(np.float32)
    want[dlogits_ref:dlogits_ref + dlogits.nbytes] = dlogits.reshape(-1).view(np.uint8)
    O.execute("port", plan.train[bwd + 1:opt], want, np.asarray(plan.rodata))
    for pid, _, g, n in info.params:
        ref = want[g:g + n * 4].view(np.float32)
        assert np.abs(ref).max() > 0
        tol.assert_close(student.arena_read(g, n * 4).view(np.float32), ref, pid)
    before = student.arena_read(0, h.persistent_size).copy()
    student.run_train_range(opt, len(plan.train))
    L.check(lib.seeml_b200_sync(C.c_void_p(student.ctx())))
    assert (student.arena_read(0, h.persistent_size) != before).any()
    student.close()
