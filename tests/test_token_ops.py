"""Vocabulary-row operators (token scores, distillation from a teacher's top entries) against
their 64-bit definitions, and their refusals."""
import ctypes as C
import math

import numpy as np
import pytest

import token_ref as R

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ---- refusals that need no device ------------------------------------------------------------
def _rc(fn, d):
    from see_ml_b200 import _lib as L
    return getattr(L.lib(), fn)(C.byref(d) if d is not None else None, None), L.last_error()


def _scores(**kw):
    from see_ml_b200 import _lib as L
    base = dict(logits=1024, labels=1024, logprob=1024, entropy=1024, stats=1024, top_logprob=1024, top_id=1024, rows=2,
                vocab=64, row_stride=64, dtype=0, top_k=4, temperature=1.0, reserved=0)
    return L.TokenScores(**{**base, **kw})


def _scores_grad(**kw):
    from see_ml_b200 import _lib as L
    base = dict(logits=1024, labels=1024, stats=1024, entropy=1024, dlogprob=1024, dentropy=1024, dlogits=1024, rows=2,
                vocab=64, row_stride=64, grad_stride=64, dtype=0, temperature=1.0)
    return L.TokenScoresGrad(**{**base, **kw})


def _distill(**kw):
    from see_ml_b200 import _lib as L
    base = dict(logits=1024, teacher_id=1024, teacher_logprob=1024, row_weight=1024, row_loss=1024, loss=1024, saved=1024,
                dlogits=1024, rows=2, vocab=64, row_stride=64, grad_stride=64, dtype=0, teacher_dtype=0, top_k=4, tail=0,
                temperature=1.0, scale=1.0)
    return L.DistillTopk(**{**base, **kw})


def _distill_grad(**kw):
    from see_ml_b200 import _lib as L
    base = dict(logits=1024, teacher_id=1024, teacher_logprob=1024, saved=1024, drow_loss=1024, dlogits=1024, rows=2,
                vocab=64, row_stride=64, grad_stride=64, dtype=0, teacher_dtype=0, top_k=4, tail=0, temperature=1.0, reserved=0)
    return L.DistillTopkGrad(**{**base, **kw})


MATRIX = [(dict(dtype=3), "unknown dtype"), (dict(vocab=0), "empty vocabulary"), (dict(rows=(1 << 27) + 1), "2^27 rows"),
          (dict(vocab=393217, row_stride=400000), "at most 393216"), (dict(row_stride=63), "row stride"),
          (dict(dtype=1, vocab=786433, row_stride=800000), "at most 786432"),
          (dict(row_stride=1 << 58), "row stride"), (dict(rows=1 << 27, vocab=1 << 16, row_stride=1 << 16), "2^44 bytes"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
          (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"),
          (dict(temperature=1e-45), "temperature"), (dict(logits=None), "logits is null"), (dict(logits=4098), "logits is not aligned")]
GRADIENT = [(dict(grad_stride=63), "gradient stride"), (dict(grad_stride=1 << 58), "gradient stride"),
            (dict(dlogits=1028), "overlaps"), (dict(dlogits=1024 + 252, row_stride=127, grad_stride=127), "overlaps"),
            (dict(grad_stride=65), "overlaps"), (dict(dlogits=1024 + 256), "overlaps")]
TEACHER = [(dict(top_k=0), "top_k"), (dict(top_k=129), "top_k"), (dict(teacher_dtype=3), "teacher dtype"),
           (dict(teacher_id=None), "teacher_id is null"), (dict(teacher_logprob=None), "teacher_logprob is null")]
REFUSED = (
    [("seeml_b200_token_scores_fwd", _scores, kw, m) for kw, m in MATRIX + [
        (dict(top_k=129), "top_k"), (dict(top_k=65), "top_k"), (dict(reserved=1), "reserved"), (dict(labels=None), "labels is null"),
        (dict(top_id=None), "top_id is null"), (dict(top_logprob=None), "top_logprob is null"),
        (dict(logprob=None, entropy=None, stats=None, top_k=0), "no output"), (dict(stats=1025), "stats is not aligned")]] +
    [("seeml_b200_token_scores_bwd", _scores_grad, kw, m) for kw, m in MATRIX + GRADIENT + [
        (dict(dlogprob=None, dentropy=None), "neither"), (dict(labels=None), "labels is null"), (dict(stats=None), "stats is null"),
        (dict(entropy=None), "entropy is null"), (dict(dlogits=None), "dlogits is null")]] +
    [("seeml_b200_distill_topk_fwd", _distill, kw, m) for kw, m in MATRIX + GRADIENT + TEACHER + [
        (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(row_loss=None), "row_loss is null")]] +
    [("seeml_b200_distill_topk_bwd", _distill_grad, kw, m) for kw, m in MATRIX + GRADIENT + TEACHER + [
        (dict(saved=None), "saved is null"), (dict(drow_loss=None), "drow_loss is null"), (dict(dlogits=None), "dlogits is null"),
        (dict(reserved=1), "reserved")]])


@pytest.mark.parametrize("fn,make,kw,message", REFUSED, ids=lambda v: None if callable(v) else str(v).replace("seeml_b200_", ""))
def test_refused_before_any_launch(backend_lib, fn, make, kw, message):
    rc, err = _rc(fn, make(**kw))
    assert rc != 0 and err.startswith("UpdateEngine: ") and message in err, err


@pytest.mark.parametrize("fn", ["seeml_b200_token_scores_fwd", "seeml_b200_token_scores_bwd", "seeml_b200_distill_topk_fwd",
                                "seeml_b200_distill_topk_bwd"])
def test_null_descriptor_is_refused(backend_lib, fn):
    rc, err = _rc(fn, None)
    assert rc != 0 and "null descriptor" in err


def test_empty_calls_need_no_device(backend_lib):
    for fn, d in (("seeml_b200_token_scores_fwd", _scores(rows=0)), ("seeml_b200_token_scores_bwd", _scores_grad(rows=0)),
                  ("seeml_b200_distill_topk_fwd", _distill(rows=0, loss=None)),
                  ("seeml_b200_distill_topk_bwd", _distill_grad(rows=0))):
        assert _rc(fn, d)[0] == 0, fn


def test_python_refuses_what_the_library_cannot_see(backend_lib):
    from see_ml_b200 import _lib as L, token_ops as T
    x = torch.zeros(4, 8)
    with pytest.raises(L.BackendError, match="device memory"):
        T.token_scores(x)
    with pytest.raises(L.BackendError, match="rows, vocab"):
        T.token_scores(torch.zeros(8))


# ---- on the device ---------------------------------------------------------------------------
def _logits(rng, rows, V, dtype, pad=0, std=3.0, masked=0.0):
    x = rng.standard_normal((rows, V)) * std
    if masked:
        hide = rng.random((rows, V)) < masked
        hide[np.arange(rows), rng.integers(0, V, rows)] = False
        x[hide] = -np.inf
    buf = torch.full((rows + 1, V + pad), 7.0, dtype=dtype, device="cuda")
    view = buf[:rows, :V]
    view.copy_(torch.from_numpy(x))
    return buf, view


def _f64(t):
    return t.double().cpu().numpy()


def _close(got, want, bound, dtype, what):
    got, want = _f64(got), np.array(want, np.float64)
    want[np.abs(want) > torch.finfo(dtype).max] *= np.inf      # beyond the type
    nonfinite = ~np.isfinite(want)
    np.testing.assert_array_equal(got[nonfinite], want[nonfinite], err_msg=what)
    err = np.abs(np.where(nonfinite, 0.0, got - np.where(nonfinite, 0.0, want)))
    bar = np.where(nonfinite, 0.0, bound + R.half_step(dtype) * np.abs(np.where(nonfinite, 0.0, want)) * (1 + 2 ** -6)) + R.floor_of(dtype)
    bad = ~(err <= bar)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} out; worst {np.max(err / bar):.3f} of the bound"


def _copies(result, rows):
    """Results of a call whose rows repeat, by copy. A row's bits depend on how it lies in the 16-byte vectors of memory,
    which repeats after 8 copies at the latest: those are returned, the others have to equal them."""
    period = 8 * rows
    out = []
    for c in range(min(8, result[1].shape[0] // rows)):
        part = []
        for t in result:
            if t is not None and t.dim():
                mine = torch.cat([t[r:r + rows] for r in range(c * rows, t.shape[0], period)])
                bits = mine.reshape(-1, rows, mine[0].numel()).contiguous().view(torch.uint8)
                assert torch.equal(bits, bits[:1].expand(bits.shape[0], -1, -1))
                t = t[c * rows:(c + 1) * rows]
            part.append(t)
        out.append(type(result)(*part))
    return out


SHAPES = [  # rows, vocab, dtype, pad, temperature, masked
    (1, 1, F32, 0, 1.0, 0.0), (3, 2, F16, 1, 0.5, 0.0), (5, 7, BF16, 0, 1.0, 0.3), (2, 33, F32, 3, 2.0, 0.5),
    (9, 255, F16, 0, 1.0, 0.0), (4, 1000, F32, 0, 0.7, 0.9), (3, 4097, BF16, 5, 1.5, 0.2), (1, 5000, F32, 0, 1.0, 0.0),
    (300, 513, F32, 0, 1.0, 0.1), (7, 32000, F32, 0, 1.0, 0.0), (2, 32000, BF16, 0, 0.8, 0.3), (5, 50001, F16, 7, 1.0, 0.0),
    (1, 131072, BF16, 0, 1.0, 0.0), (3, 100003, F32, 0, 2.0, 0.6), (2, 393216, F32, 0, 1.0, 0.0), (1, 786432, F16, 0, 1.0, 0.0),
    # calls of many rows, which give each row to one block
    (300, 1, F32, 0, 1.0, 0.0), (301, 11, BF16, 2, 1.0, 0.2), (400, 1027, F16, 0, 0.6, 0.4), (300, 9001, F32, 3, 1.0, 0.0),
    (297, 20001, BF16, 0, 1.5, 0.3), (310, 16384, F16, 8, 1.0, 0.0)]


def _ids(v):
    return str(v).replace("torch.", "")


@gpu
@pytest.mark.parametrize("rows,V,dtype,pad,T,masked", SHAPES, ids=_ids)
@pytest.mark.parametrize("k", [0, 1, 20, 128])
def test_token_scores(backend_lib, rows, V, dtype, pad, T, masked, k):
    from see_ml_b200 import token_ops as ops
    k = min(k, V)
    rng = np.random.default_rng(V * 31 + k)
    _, x = _logits(rng, rows, V, dtype, pad, masked=masked)
    labels = rng.integers(-1, V, rows).astype(np.int32)
    s = ops.token_scores(x, torch.from_numpy(labels).cuda(), top_k=k, temperature=T, stats=True)
    lp, h, tlp, tid = R.scores(_f64(x), labels, k, T)
    d = R.delta(V)
    _close(s.logprob, lp, d, F32, "logprob")
    _close(s.entropy, h, 2 * (1 + math.log(V)) * d, F32, "entropy")
    _close(s.stats[:, 0], _f64(x).max(1), 0.0, F32, "max")
    if k:
        np.testing.assert_array_equal(s.top_id.cpu().numpy(), tid)
        _close(s.top_logprob, tlp, d, F32, "top_logprob")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=_ids)
@pytest.mark.parametrize("V,k", [(40, 40), (900, 100), (1900, 128), (3000, 16), (32000, 128), (100003, 100)])
@pytest.mark.parametrize("copies", [1, 160, 1200])
@pytest.mark.parametrize("shape", ["constant", "ascending", "descending", "few", "one_slice", "zeros_of_both_signs", "lowest"])
def test_top_alternatives_of_awkward_rows(backend_lib, dtype, V, k, shape, copies):
    """Ties go to the lower index, whatever the order and wherever the great values lie."""
    if copies * V > 20000000:
        pytest.skip("more than this adds nothing: calls of so many long rows go the way of 160 copies")
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V + k)
    j = np.arange(V)
    x = {"constant": np.full(V, 1.5), "ascending": j / V * 8, "descending": -j / V * 8, "few": rng.integers(0, 3, V) * 1.0,
         "one_slice": np.where((j // 8) % 512 == 3, 5.0 + rng.standard_normal(V), rng.standard_normal(V)),
         "zeros_of_both_signs": np.where(j % 2, 0.0, -0.0), "lowest": np.full(V, torch.finfo(dtype).min)}[shape]
    t = torch.from_numpy(np.stack([x, x[::-1].copy()])).to(dtype).cuda()
    _, h, tlp, tid = R.scores(_f64(t), None, k, 1.0)
    for s in _copies(ops.token_scores(t.repeat(copies, 1), None, top_k=k), 2):
        np.testing.assert_array_equal(s.top_id.cpu().numpy(), tid)
        _close(s.top_logprob, tlp, R.delta(V), F32, "top_logprob")
        _close(s.entropy, h, 2 * (1 + math.log(V)) * R.delta(V), F32, "entropy")


@gpu
@pytest.mark.parametrize("copies", [1, 43])
@pytest.mark.parametrize("V", [5, 700, 32000])
def test_rows_that_are_masked_or_not_finite(backend_lib, V, copies):
    from see_ml_b200 import token_ops as ops
    x = np.random.default_rng(V).standard_normal((7, V))
    x[0] = -np.inf                           # nothing left
    x[1, 2] = np.nan
    x[2, 3] = np.inf
    x[3, 1:] = -np.inf                       # one token left
    x[4, ::2] = -3.4e38
    x[5, 1] = np.nan
    x[5, 4] = np.nan
    t = torch.from_numpy(x).float().cuda()
    labels = np.array([1, 0, 0, 0, 1, 3, V + 5], np.int32)
    lp, h, tlp, tid = R.scores(_f64(t), labels, 4, 0.5)
    for s in _copies(ops.token_scores(t.repeat(copies, 1), torch.from_numpy(labels).cuda().repeat(copies), top_k=4,
                                      temperature=0.5, stats=True), 7):
        np.testing.assert_array_equal(s.top_id.cpu().numpy(), tid)
        _close(s.logprob, lp, R.delta(V), F32, "logprob")
        _close(s.entropy, h, 2 * (1 + math.log(V)) * R.delta(V), F32, "entropy")
        _close(s.top_logprob, tlp, R.delta(V), F32, "top_logprob")
    ones = torch.ones(7, device="cuda")
    g = _f64(ops.token_scores_backward(t, torch.from_numpy(labels).cuda(), s.stats, s.entropy, ones, ones, temperature=0.5))
    assert (g[0] == 0).all() and np.isnan(g[1]).all() and np.isnan(g[2]).all() and np.isnan(g[6]).all()
    assert (g[3] == 0).all() and np.isfinite(g[4]).all() and np.isnan(g[5]).all()


@gpu
@pytest.mark.parametrize("rows,V,dtype,pad,T,masked", SHAPES, ids=_ids)
@pytest.mark.parametrize("parts", ["both", "logprob", "entropy"])
def test_token_scores_gradient(backend_lib, rows, V, dtype, pad, T, masked, parts):
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V * 7 + rows)
    _, x = _logits(rng, rows, V, dtype, pad, masked=masked)
    labels = rng.integers(-1, V, rows).astype(np.int32)
    gl, gh = rng.standard_normal((2, rows)).astype(np.float32)
    gl[rows // 2] = gh[rows // 2] = 0.0
    lab = torch.from_numpy(labels).cuda()
    s = ops.token_scores(x, lab, temperature=T, stats=True)
    up = [torch.from_numpy(v).cuda() for v in (gl, gh)]
    g = ops.token_scores_backward(x, lab, s.stats, s.entropy, up[0] if parts != "entropy" else None,
                                  up[1] if parts != "logprob" else None, temperature=T)
    want, err = R.scores_grad(_f64(x), labels, gl.astype(np.float64) * (parts != "entropy"),
                              gh.astype(np.float64) * (parts != "logprob"), T)
    _close(g, want, err, dtype, "dlogits")


def _teacher(rng, rows, V, K, dtype, absent=0.0):
    ids = np.stack([rng.permutation(V)[:K] if V < 200000 else np.unique(rng.integers(0, V, 4 * K))[:K] for _ in range(rows)])
    if K > V:
        ids = np.concatenate([ids, np.full((rows, K - V), -1)], 1)
    v = rng.standard_normal((rows, K)) * 1.5
    v = v - np.log(np.exp(v).sum(1, keepdims=True)) + math.log(0.9)
    ids = np.where(rng.random((rows, K)) < absent, -1, ids).astype(np.int32)
    return torch.from_numpy(ids).cuda(), torch.from_numpy(v).to(dtype).cuda()


@gpu
@pytest.mark.parametrize("rows,V,dtype,pad,T,masked", SHAPES, ids=_ids)
@pytest.mark.parametrize("K,tail,tdtype", [(1, True, F32), (17, False, BF16), (128, True, F16), (33, True, F32)], ids=_ids)
def test_distill(backend_lib, rows, V, dtype, pad, T, masked, K, tail, tdtype):
    """Loss, its gradient in the same pass, and the gradient of a pass of its own."""
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V * 13 + K)
    buf, x = _logits(rng, rows, V, dtype, pad, masked=masked if K < 17 else 0.0)
    ids, v = _teacher(rng, rows, V, K, tdtype, absent=0.1)
    if masked and K < 17:        # a masked token that the teacher names makes the loss infinite
        x.scatter_(1, ids.clamp(min=0).long(), 1.0)
    before = buf.clone()
    w = rng.integers(0, 3, rows).astype(np.float32)
    scale = 0.25
    wt = torch.from_numpy(w).cuda()
    r = ops.distill_topk(x, ids, v, row_weight=wt, scale=scale, temperature=T, tail=tail, grad=True, saved=True)
    loss, lerr, grad, gerr = R.distill(_f64(x), ids.cpu().numpy(), _f64(v), T, tail)
    loss, lerr = np.where(w == 0, 0.0, loss), np.where(w == 0, 0.0, lerr)
    _close(r.row_loss, loss, lerr, F32, "row_loss")
    _close(r.loss, scale * (w * loss).sum(), scale * (w * (lerr + np.abs(loss) * R.U)).sum(), F32, "loss")
    up = (scale * w.astype(np.float64))[:, None]
    _close(r.dlogits, grad * up, gerr * up, dtype, "dlogits")
    d = torch.from_numpy((w * scale).astype(np.float32)).cuda()
    g = ops.distill_topk_backward(x, ids, v, r.saved, d, temperature=T, tail=tail)
    _close(g, grad * up, gerr * up, dtype, "dlogits of the backward call")
    assert torch.equal(buf, before)
    alone = ops.distill_topk(x, ids, v, row_weight=wt, scale=scale, temperature=T, tail=tail)
    _close(alone.row_loss, loss, lerr, F32, "row_loss alone")
    _close(alone.loss, scale * (w * loss).sum(), scale * (w * (lerr + np.abs(loss) * R.U)).sum(), F32, "loss alone")
    inplace = ops.distill_topk(x, ids, v, row_weight=wt, scale=scale, temperature=T, tail=tail, out=x)
    assert inplace.dlogits is x and torch.equal(x, r.dlogits) and torch.equal(inplace.row_loss, r.row_loss)
    assert torch.equal(buf[rows], before[rows]) and torch.equal(buf[:, V:], before[:, V:])


@gpu
@pytest.mark.parametrize("copies", [1, 30])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [9, 3000, 70001, 140003])
def test_distill_of_awkward_rows(backend_lib, V, tail, copies):
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V)
    x = rng.standard_normal((10, V)) * 2
    ids = np.stack([rng.permutation(V)[:6] for _ in range(10)]).astype(np.int32)
    v = np.log(np.tile([0.4, 0.2, 0.1, 0.1, 0.05, 0.05], (10, 1)))
    ids[0] = -1                       # no entry
    v[1] = -np.inf                    # entries without mass
    ids[2] = ids[2, 0]                # one token named by all
    ids[3, 4] = ids[3, 1]             # and by two
    v[4, 2] = -np.inf                 # a named token without mass
    x[5] = -np.inf                    # nothing left of the student
    x[6, ids[6, 3]] = -np.inf         # the student masks a token that the teacher wants
    ids[7, 0] = V                     # beyond the vocabulary
    x[8] = -300.0                     # the unnamed tokens vanish beside the named ones in f32
    x[8, ids[8]] = 20.0
    ids[9, 3:] = -1
    t = torch.from_numpy(x).float().cuda()
    vt = torch.from_numpy(v).float().cuda()
    it = torch.from_numpy(ids).cuda()
    good = [i for i in range(10) if i != 7]
    for out in (None, t.repeat(copies, 1)):
        src = t.repeat(copies, 1) if out is None else out
        loss, lerr, grad, gerr = R.distill(_f64(t)[good], ids[good], _f64(vt)[good], 1.0, tail)
        for r in _copies(ops.distill_topk(src, it.repeat(copies, 1), vt.repeat(copies, 1), tail=tail, grad=True, saved=True,
                                          out=out), 10):
            _close(r.row_loss[good], loss, lerr, F32, "row_loss")
            _close(r.dlogits[good], grad, gerr, F32, "dlogits")
            assert torch.isnan(r.row_loss[7]) and torch.isnan(r.dlogits[7]).all()
    g = ops.distill_topk_backward(t, it, vt, r.saved.contiguous(), torch.ones(10, device="cuda"), tail=tail)
    _close(g[good], grad, gerr, F32, "dlogits of the backward call")
    assert torch.isnan(g[7]).all()
    x[5, 0] = np.nan                  # a row of weight 0 is not looked at, another is
    t = torch.from_numpy(x).float().cuda()
    w = torch.ones(10, device="cuda")

    def weighted():
        return _copies(ops.distill_topk(t.repeat(copies, 1), it.repeat(copies, 1), vt.repeat(copies, 1), tail=tail, grad=True,
                                        row_weight=w.repeat(copies)), 10)[0]
    r = weighted()
    assert torch.isnan(r.row_loss[5]) and torch.isnan(r.dlogits[5]).all() and torch.isnan(r.loss)
    w[5] = w[6] = w[7] = 0.0
    r = weighted()
    assert (r.row_loss[5:8] == 0).all() and (r.dlogits[5:8] == 0).all() and torch.isfinite(r.loss)


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_gradients_against_differences(backend_lib, tail):
    """Central differences of the kernels' own losses: truncation h^2 / 6 |f'''| <= h^2 / T^3, rounding of the two
    values delta / h each."""
    from see_ml_b200 import token_ops as ops
    V, T, h = 37, 1.3, 2.0 ** -6
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((1, V))).float().cuda()
    steps = torch.cat([x + h * torch.eye(V, device="cuda"), x - h * torch.eye(V, device="cuda")])
    width = (steps[:V] - steps[V:]).diagonal()
    ids, v = _teacher(rng, 1, V, 6, F32)
    r = ops.distill_topk(x, ids, v, temperature=T, tail=tail, grad=True)
    f = ops.distill_topk(steps, ids.expand(2 * V, -1).contiguous(), v.expand(2 * V, -1).contiguous(), temperature=T, tail=tail).row_loss
    lab = torch.tensor([4], dtype=torch.int32, device="cuda")
    s = ops.token_scores(x, lab, temperature=T, stats=True)
    one = torch.ones(1, device="cuda")
    g = ops.token_scores_backward(x, lab, s.stats, s.entropy, one, -one, temperature=T)
    f2 = ops.token_scores(steps, lab.expand(2 * V).contiguous(), temperature=T)
    bar = h * h / T ** 3 * (2 + math.log(V)) + 2 * (2 + 2 * math.log(V)) * R.delta(V) / h
    assert ((f[:V] - f[V:]) / width - r.dlogits[0]).abs().max().item() <= bar
    f2 = f2.logprob - f2.entropy
    assert ((f2[:V] - f2[V:]) / width - g[0]).abs().max().item() <= bar


@gpu
@pytest.mark.parametrize("dtype,V", [(BF16, 4097), (F32, 1000), (F16, 32001), (F32, 35003)], ids=_ids)
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("xo,go,xs,gs", [(0, 0, 0, 0), (1, 0, 3, 0), (0, 5, 0, 8), (3, 3, 7, 7), (8, 2, 1, 9)])
def test_alignments_and_strides(backend_lib, dtype, V, xo, go, xs, gs, rows):
    """Rows that start anywhere, gradients whose rows start elsewhere; nothing beside them is touched."""
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V + xo)
    xb = torch.zeros(16 + rows * (V + xs), dtype=dtype, device="cuda")
    x = xb[xo:xo + rows * (V + xs)].view(rows, V + xs)[:, :V]
    x.copy_(torch.from_numpy(rng.standard_normal((rows, V)) * 2))
    gb = torch.full((16 + rows * (V + gs),), 3.0, dtype=dtype, device="cuda")
    g = gb[go:go + rows * (V + gs)].view(rows, V + gs)[:, :V]
    ids, v = _teacher(rng, rows, V, 128, F32)
    lab = torch.arange(rows, dtype=torch.int32, device="cuda") * (V // rows) + torch.arange(rows, dtype=torch.int32, device="cuda") % 8
    lab.clamp_(max=V - 1)
    one = torch.ones(rows, device="cuda")
    flat = x.contiguous()
    s0, s1 = ops.token_scores(flat, lab, top_k=9), ops.token_scores(x, lab, top_k=9, stats=True)
    assert torch.equal(s0.top_id, s1.top_id)
    _close(s1.logprob, _f64(s0.logprob), 2 * R.delta(V), F32, "logprob")
    loss, lerr, grad, gerr = R.distill(_f64(x), ids.cpu().numpy(), _f64(v), 1.0, True)
    r = ops.distill_topk(x, ids, v, tail=True, out=g, saved=True)
    _close(r.row_loss, loss, lerr, F32, "row_loss")
    for call in (lambda: None, lambda: ops.distill_topk_backward(x, ids, v, r.saved, one, tail=True, out=g.zero_())):
        call()
        _close(g, grad, gerr, dtype, "dlogits")
        edge = gb.clone()
        edge[go:go + rows * (V + gs)].view(rows, V + gs)[:, :V] = 3.0
        assert (edge == 3.0).all()
    want, err = R.scores_grad(_f64(x), lab.cpu().numpy(), np.ones(rows), -np.ones(rows), 1.0)
    ops.token_scores_backward(x, lab, s1.stats, s1.entropy, one, -one, out=g.zero_())
    _close(g, want, err, dtype, "dlogits of the scores")


@gpu
@pytest.mark.parametrize("dtype,off", [(BF16, 3), (F16, 8), (F32, 1), (BF16, 0)], ids=_ids)
@pytest.mark.parametrize("V", [17000, 70003])
def test_every_token_once_named_and_once_the_label(backend_lib, dtype, off, V):
    """A row per window of tokens: each token's own gradient survives whichever block writes beside it."""
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V)
    K = 128
    rows = -(-V // K)
    xb = torch.zeros(rows * V + 16, dtype=dtype, device="cuda")
    x = xb[off:off + rows * V].view(rows, V)
    x.copy_(torch.randn(V, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") * 2)
    ids = (torch.arange(rows * K, device="cuda", dtype=torch.int32).view(rows, K)) % V
    v = torch.full((rows, K), -math.log(K / 0.875), device="cuda")
    p = torch.softmax(x[:1].double(), 1)
    target = torch.zeros(rows, V, dtype=torch.float64, device="cuda").scatter_add_(1, ids.long(), v.double().exp())
    named = torch.zeros(rows, V, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), True)
    tail = torch.where(named, 0.0, p).sum(1, keepdim=True)
    want = p - target - torch.where(named, 0.0, 0.125 * p / tail)
    bound = 4 * R.delta(V) * (p + 0.125 * p / tail) + 8 * R.U * target + R.half_step(dtype) * want.abs() * (1 + 2 ** -6) + R.floor_of(dtype)
    r = ops.distill_topk(x, ids, v, tail=True, grad=True, saved=True)
    assert ((r.dlogits - want).abs() <= bound).all()
    g = ops.distill_topk_backward(x, ids, v, r.saved, torch.ones(rows, device="cuda"), tail=True)
    assert ((g - want).abs() <= bound).all()
    lab = torch.arange(rows, device="cuda", dtype=torch.int32)
    up = torch.ones(rows, device="cuda")
    for first in range(0, V, max(1, rows * 7)):
        lab = (torch.arange(rows, device="cuda", dtype=torch.int32) * 7 + first) % V
        s = ops.token_scores(x, lab, stats=True)
        want = -p.expand(rows, -1).clone()
        want.scatter_add_(1, lab.long()[:, None], torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
        got = ops.token_scores_backward(x, lab, s.stats, s.entropy, up, None)
        bound = 4 * R.delta(V) * p + 4 * R.U + R.half_step(dtype) * want.abs() * (1 + 2 ** -6) + R.floor_of(dtype)
        assert ((got - want).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dtype,off", [(BF16, 3), (F16, 8), (F32, 1), (F32, 0)], ids=_ids)
@pytest.mark.parametrize("V", [40, 4500])
def test_scores_gradient_of_many_rows(backend_lib, dtype, off, V):
    """Every token once the label, in as many rows; rows without an upstream gradient among them."""
    from see_ml_b200 import token_ops as ops
    rows = max(V, 1000)
    gen = torch.Generator(device="cuda").manual_seed(V)
    xb = torch.zeros(rows * V + 16, dtype=dtype, device="cuda")
    x = xb[off:off + rows * V].view(rows, V)
    x.copy_(torch.randn(rows, V, generator=gen, device="cuda") * 2)
    lab = torch.arange(rows, device="cuda", dtype=torch.int32) % V
    gl = torch.randn(rows, generator=gen, device="cuda")
    gl[::7] = 0.0
    s = ops.token_scores(x, lab, stats=True)
    p = torch.softmax(x.double(), 1)
    one = torch.zeros_like(p).scatter_(1, lab.long()[:, None], 1.0)
    want = gl.double()[:, None] * (one - p)
    bound = gl.double().abs()[:, None] * (4 * R.delta(V) * p + 4 * R.U * one) + R.half_step(dtype) * want.abs() * (1 + 2 ** -6) + R.floor_of(dtype)
    got = ops.token_scores_backward(x, lab, s.stats, s.entropy, gl, None)
    assert ((got - want).abs() <= bound).all()
    inplace = ops.token_scores_backward(x, lab, s.stats, s.entropy, gl, None, out=x)
    assert inplace is x and torch.equal(x, got) and (xb[:off] == 0).all() and (xb[off + rows * V:] == 0).all()


@gpu
def test_rows_beyond_32_bits_of_offset(backend_lib):
    from see_ml_b200 import token_ops as ops
    rows, V, stride = 3, 1001, (1 << 31) + 8
    buf = torch.empty(2 * stride + V, dtype=BF16, device="cuda")
    x = buf.as_strided((rows, V), (stride, 1))
    rng = np.random.default_rng(0)
    x.copy_(torch.from_numpy(rng.standard_normal((rows, V)) * 2))
    flat = x.contiguous()
    lab = torch.arange(rows, dtype=torch.int32, device="cuda")
    ids, v = _teacher(rng, rows, V, 5, F32)
    a, b = ops.token_scores(x, lab, top_k=5), ops.token_scores(flat, lab, top_k=5)
    assert torch.equal(a.top_id, b.top_id)
    _close(a.logprob, _f64(b.logprob), 2 * R.delta(V), F32, "logprob")
    _, _, grad, gerr = R.distill(_f64(flat), ids.cpu().numpy(), _f64(v), 1.0, True)
    ops.distill_topk(x, ids, v, tail=True, out=x)
    _close(x, grad, gerr, BF16, "dlogits in place")


@gpu
@pytest.mark.parametrize("V", [1, 3, 10])
def test_a_million_rows_of_a_small_vocabulary(backend_lib, V):
    """Against the same formulas in 64 bits on the device; the entries name the first and the last token. Bounds: twice
    delta, for values up to 16."""
    from see_ml_b200 import token_ops as ops
    rows = 1000003
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(rows, V, generator=g, device="cuda") * 2
    lab = torch.randint(V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    s = ops.token_scores(x, lab, top_k=1, stats=True)
    lp = torch.log_softmax(x.double(), 1)
    p = lp.exp()
    H = -(p * lp).sum(1)
    d = R.delta(V) * 2
    assert (s.logprob - lp.gather(1, lab.long()[:, None])[:, 0]).abs().max() <= d * 16
    assert (s.entropy - H).abs().max() <= d * 16
    assert torch.equal(s.top_id[:, 0].long(), x.argmax(1))
    up = torch.ones(rows, device="cuda")
    got = ops.token_scores_backward(x, lab, s.stats, s.entropy, up, None)
    want = torch.zeros_like(p).scatter_(1, lab.long()[:, None], 1.0) - p
    assert (got - want).abs().max() <= d * 16
    ids = torch.tensor([[0, V - 1]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
    q = torch.tensor([[0.5, 0.25]], device="cuda").expand(rows, 2)
    r = ops.distill_topk(x, ids, q.log().contiguous(), tail=True, grad=True, scale=1.0, saved=True)
    target = torch.zeros_like(p).scatter_add_(1, ids.long(), q.double())
    named = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids.long(), True)
    tail = torch.where(named, 0.0, p).sum(1, keepdim=True)
    rest = 0.25 if V > 2 else 0.0                         # with every token named the tail's term is left out
    want = p * (0.75 + rest) - target - torch.where(named, 0.0, p * rest / tail.clamp(min=1e-300))
    assert (r.dlogits - want).abs().max() <= d * 16
    again = ops.distill_topk_backward(x, ids, q.log().contiguous(), r.saved, up, tail=True)
    assert (again - want).abs().max() <= d * 16
    loss = (q.double() * (q.double().log() - lp.gather(1, ids.long()))).sum(1)
    if V > 2:
        loss += rest * (math.log(rest) - tail[:, 0].log())
    assert (r.row_loss - loss).abs().max() <= d * 16
    assert abs(r.loss.item() - loss.sum().item()) <= rows * d * 16


@gpu
def test_interleaved_gradient_rows(backend_lib):
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(3)
    both = torch.zeros(6, 2 * 500, device="cuda")
    x, g = both[:, :500], both[:, 500:]
    x.copy_(torch.from_numpy(rng.standard_normal((6, 500))))
    ids, v = _teacher(rng, 6, 500, 4, F32)
    _, _, grad, gerr = R.distill(_f64(x), ids.cpu().numpy(), _f64(v), 1.0, False)
    _close(ops.distill_topk(x, ids, v, out=g).dlogits, grad, gerr, F32, "dlogits")


@gpu
def test_device_refusals(backend_lib):
    from see_ml_b200 import _lib as L, token_ops as ops
    x = torch.zeros(4, 64, device="cuda")
    ids, v = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    for bad in (lambda: ops.token_scores(x.double()), lambda: ops.token_scores(x.t()), lambda: ops.token_scores(x[:1].expand(4, -1)),
                lambda: ops.token_scores(x, torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: ops.token_scores(x, torch.zeros(4, dtype=torch.int32)), lambda: ops.token_scores(x, top_k=65),
                lambda: ops.token_scores(x, temperature=0.0), lambda: ops.distill_topk(x, ids.long(), v),
                lambda: ops.distill_topk(x, ids[:3], v), lambda: ops.distill_topk(x, ids, v, out=x.half()),
                lambda: ops.distill_topk(x, ids, v.t().contiguous().t()), lambda: ops.distill_topk(x, ids, v, scale=math.inf),
                lambda: ops.distill_topk(x[:, :32], ids, v, out=x[:, 1:33]),
                lambda: ops.distill_topk(x, ids, None)):
        with pytest.raises(L.BackendError, match="^UpdateEngine: "):
            bad()
    host = np.zeros(256, np.float32)
    rc, err = _rc("seeml_b200_token_scores_fwd", _scores(logits=x.data_ptr(), labels=host.ctypes.data, top_k=0, entropy=None,
                                                         stats=None, logprob=v.data_ptr()))
    assert rc != 0 and "labels" in err
    empty = ops.distill_topk(x[:0], ids[:0], v[:0], grad=True)
    assert empty.loss.item() == 0.0 and empty.dlogits.shape == (0, 64)
    assert ops.token_scores(x[:0], ids[:0, 0], top_k=3).top_id.shape == (0, 3)


@gpu
@pytest.mark.parametrize("rows", [40, 320])
def test_streams_and_graphs_give_the_same_bits(backend_lib, rows):
    """The calls of a step on two streams at once and in two captured graphs: no scratch is shared."""
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(1)
    V, k = 20011, 24
    xs = [torch.from_numpy(rng.standard_normal((rows, V)) * 2).to(BF16).cuda() for _ in range(2)]
    lab = torch.arange(rows, dtype=torch.int32, device="cuda")
    one = torch.ones(rows, device="cuda")

    def step(teacher, student):
        s = ops.token_scores(teacher, lab, top_k=k, stats=True)
        r = ops.distill_topk(student, s.top_id, s.top_logprob, scale=1 / rows, tail=True, grad=True)
        g = ops.token_scores_backward(teacher, lab, s.stats, s.entropy, one, -one)
        return [s.logprob, s.entropy, s.top_id, s.top_logprob, r.loss, r.row_loss, r.dlogits, g]

    want = [[t.clone() for t in step(xs[0], xs[1])], [t.clone() for t in step(xs[1], xs[0])]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = step(xs[i], xs[1 - i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(xs[i], xs[1 - i]))
        graphs.append(g)
    for _ in range(2):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    a, b = xs[0].clone(), xs[1].clone()
    xs[0].copy_(b)
    xs[1].copy_(a)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want[1], outs[0]))


@gpu
@pytest.mark.parametrize("dtype,V", [(F32, 40), (BF16, 700), (F16, 3001), (F32, 20003), (BF16, 140003)], ids=_ids)
@pytest.mark.parametrize("copies", [1, 100])
@pytest.mark.parametrize("tail", [False, True])
def test_backward_of_rows_that_the_forward_call_skipped(backend_lib, dtype, V, copies, tail):
    """A row of weight 0 has a loss of 0 whatever its logits and entries, so its gradient is 0 whatever comes from above."""
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V)
    x = rng.standard_normal((3, V))
    x[0] += 200.0                     # exp(x / T) is beyond f32
    x[1, 1], x[1, 2] = np.nan, np.inf
    t = torch.from_numpy(x).to(dtype).cuda()
    ids, v = _teacher(rng, 3, V, 5, F32)
    ids[1, 0] = V                     # beyond the vocabulary
    w, up = torch.tensor([0.0, 0.0, 1.0], device="cuda"), torch.tensor([1.0, -2.0, 3.0], device="cuda")
    _, _, grad, gerr = R.distill(_f64(t)[2:], ids.cpu().numpy()[2:], _f64(v)[2:], 0.5, tail)
    many = [a.repeat(copies, *[1] * (a.dim() - 1)) for a in (t, ids, v, w, up)]
    r = ops.distill_topk(*many[:3], row_weight=many[3], temperature=0.5, tail=tail, saved=True)
    for out in (None, torch.empty(3 * copies, V + 1, dtype=dtype, device="cuda")[:, 1:]):
        g = ops.distill_topk_backward(*many[:3], r.saved, many[4], temperature=0.5, tail=tail, out=out).view(copies, 3, V)
        assert (g[:, :2] == 0).all()
        for c in {0, copies // 2, copies - 1}:
            _close(g[c, 2:], 3.0 * grad, 3.0 * gerr, dtype, "dlogits of a row that counted")


@gpu
@pytest.mark.parametrize("rows,V", [(6, 9), (6, 3000), (6, 140003), (300, 9), (300, 3500), (300, 30000), (300, 140003)])
@pytest.mark.parametrize("tail", [False, True])
def test_row_that_is_not_finite_has_no_loss_without_a_teacher_either(backend_lib, rows, V, tail):
    """Entries that are absent, or without mass, leave neither the loss nor the gradient of such a row finite."""
    from see_ml_b200 import token_ops as ops
    x = torch.zeros(rows, V, device="cuda")
    x[0::6, 3], x[1::6, 4], x[2::6, 0] = math.nan, math.inf, math.nan
    ids = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    ids[2::6, 1] = ids[3::6, 0] = 0                           # the token itself, named without mass
    v = torch.full((rows, 2), -math.inf, device="cuda")
    r = ops.distill_topk(x, ids, v, tail=tail, grad=True, saved=True)
    alone = ops.distill_topk(x, ids, v, tail=tail)
    g = ops.distill_topk_backward(x, ids, v, r.saved, torch.ones(rows, device="cuda"), tail=tail)
    lost = torch.arange(rows, device="cuda") % 6 < 3
    for loss in (r.row_loss, alone.row_loss):
        assert loss[lost].isnan().all() and loss[~lost].isfinite().all()
    assert r.loss.isnan() and alone.loss.isnan()
    for d in (r.dlogits, g):
        assert d[lost].isnan().all() and d[~lost].isfinite().all()


COLD = np.float32(1e-30)                                      # the lowest temperature that is taken


@pytest.mark.parametrize("fn,make", [("seeml_b200_token_scores_fwd", _scores), ("seeml_b200_token_scores_bwd", _scores_grad),
                                     ("seeml_b200_distill_topk_fwd", _distill), ("seeml_b200_distill_topk_bwd", _distill_grad)],
                         ids=lambda v: v.replace("seeml_b200_", "") if isinstance(v, str) else "")
def test_temperatures_next_to_the_lowest(backend_lib, fn, make):
    """Below it log2(e) / T and the gradients' factors leave f32; 3.5e-39 has a finite 1 / T and no finite log2(e) / T."""
    for t in (np.nextafter(COLD, np.float32(0)), 3.5e-39, 1e-38):
        rc, err = _rc(fn, make(temperature=t))
        assert rc != 0 and "temperature" in err, (t, err)
    for t in (COLD, 3e38):
        assert _rc(fn, make(temperature=t, rows=0, **({"loss": None} if make is _distill else {})))[0] == 0


@gpu
@pytest.mark.parametrize("rows", [2, 400])
def test_the_lowest_temperature(backend_lib, rows):
    """p is 1 / 2 on the two greatest tokens and 0 elsewhere, exactly; gradients are those of T = 1 over T."""
    from see_ml_b200 import token_ops as ops
    V, T = 5000, float(COLD)
    x = torch.zeros(rows, V, device="cuda")
    x[:, 7] = x[:, 4000] = 2.0
    x[:, 100:200] = -math.inf
    lab = torch.full((rows,), 7, dtype=torch.int32, device="cuda")
    s = ops.token_scores(x, lab, top_k=3, temperature=T, stats=True)
    half = abs(math.log(0.5))
    assert ((s.logprob + half).abs() <= 4 * R.U).all() and ((s.entropy - half).abs() <= 4 * R.U).all()
    assert s.top_id[:, 0].eq(7).all() and s.top_id[:, 1].eq(4000).all() and s.top_logprob[:, 2].lt(-1e30).all()
    one = torch.ones(rows, device="cuda")
    want = torch.zeros(rows, V, dtype=torch.float64, device="cuda")
    want[:, 7], want[:, 4000] = 0.5 / T, -0.5 / T
    got = ops.token_scores_backward(x, lab, s.stats, s.entropy, one, None, temperature=T)
    assert ((got - want).abs() <= 8 * R.U / T).all() and (got[:, 100:200] == 0).all()
    got = ops.token_scores_backward(x, lab, s.stats, s.entropy, None, one, temperature=T)      # H is at its greatest
    assert (got.abs() <= 8 * R.U / T).all() and (got[:, 100:200] == 0).all()
    ids = torch.tensor([[7, 0]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
    v = torch.tensor([[-half, -math.inf]], device="cuda").expand(rows, 2).contiguous()
    want[:, 7], want[:, 4000] = 0.0, 0.0                       # p is the teacher's: half on 7, the rest on 4000
    r = ops.distill_topk(x, ids, v, temperature=T, tail=True, grad=True, saved=True)
    g = ops.distill_topk_backward(x, ids, v, r.saved, one, temperature=T, tail=True)
    assert (r.row_loss.abs() <= 8 * R.U).all()
    for d in (r.dlogits, g):
        assert (d.abs() <= 8 * R.U / T).all() and (d[:, 100:200] == 0).all()


@gpu
def test_gradients_written_in_place_count_as_modifications(backend_lib):
    """A node that kept the logits for its own backward pass does not compute with what the gradient left there."""
    from see_ml_b200 import token_ops as ops
    lab, one = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda")
    ids, v = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, 1, device="cuda")
    x = torch.zeros(4, 64, device="cuda")
    s, r = ops.token_scores(x, lab, stats=True), ops.distill_topk(x, ids, v, saved=True)
    for write in (lambda z: ops.token_scores_backward(z, lab, s.stats, s.entropy, one, None, out=z),
                  lambda z: ops.distill_topk(z, ids, v, out=z),
                  lambda z: ops.distill_topk_backward(z, ids, v, r.saved, one, out=z)):
        leaf = torch.zeros(4, 64, device="cuda", requires_grad=True)
        z = leaf + 1.0
        loss = (z * z).sum()                                  # keeps z
        before = z._version
        write(z)
        assert z._version > before
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
        with torch.inference_mode():                          # such tensors have no counter
            write(torch.zeros(4, 64, device="cuda"))
    before = x._version
    ops.distill_topk(x, ids, v, grad=True)
    assert x._version == before                               # a gradient of its own leaves the logits alone


# rows of 4 to 16 KiB of many rows go to a warp each, of few rows to blocks; both sides of the streamed kernels
NOT_FINITE = [(F32, 2000), (BF16, 5000), (F16, 7001), (BF16, 40), (F16, 20011), (F32, 9001)]


@gpu
@pytest.mark.parametrize("dtype,V", NOT_FINITE, ids=_ids)
@pytest.mark.parametrize("copies,k", [(1, 4), (43, 2), (343, 16)])
def test_scores_of_rows_that_are_not_finite(backend_lib, dtype, V, copies, k):
    from see_ml_b200 import token_ops as ops
    x = np.random.default_rng(V).standard_normal((8, V))
    low = float(torch.finfo(dtype).min)
    x[0] = -np.inf
    x[1, V // 2] = np.nan
    x[2, V - 1] = np.inf
    x[3, 1:] = -np.inf
    x[4, ::2] = low
    x[5] = low
    x[6, 1], x[6, V - 2], x[6, 3] = np.nan, np.nan, np.inf
    t = torch.from_numpy(x).to(dtype).cuda()
    labels = np.array([1, 0, 0, 0, 1, 3, 2, V], np.int32)
    lab = torch.from_numpy(labels).cuda()
    lp, h, tlp, tid = R.scores(_f64(t), labels, k, 0.5)
    for s in _copies(ops.token_scores(t.repeat(copies, 1), lab.repeat(copies), top_k=k, temperature=0.5, stats=True), 8):
        np.testing.assert_array_equal(s.top_id.cpu().numpy(), tid)
        _close(s.logprob, lp, R.delta(V), F32, "logprob")
        _close(s.entropy, h, 2 * (1 + math.log(V)) * R.delta(V), F32, "entropy")
        _close(s.top_logprob, tlp, R.delta(V), F32, "top_logprob")
    up = torch.ones(8 * copies, device="cuda")
    many, stats, ent = t.repeat(copies, 1), s.stats.repeat(copies, 1), s.entropy.repeat(copies)
    g = ops.token_scores_backward(many, lab.repeat(copies), stats, ent, up, up, temperature=0.5).view(copies, 8, V)
    assert (g[:, 0] == 0).all() and g[:, [1, 2, 6, 7]].isnan().all() and (g[:, 3] == 0).all()
    want, err = R.scores_grad(_f64(t)[4:6], labels[4:6], np.ones(2), np.ones(2), 0.5)
    for c in {0, copies // 2, copies - 1}:
        _close(g[c, 4:6], want, err, dtype, "dlogits")


@gpu
@pytest.mark.parametrize("dtype,V", NOT_FINITE + [(BF16, 140003)], ids=_ids)
@pytest.mark.parametrize("copies", [1, 43])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_of_rows_that_are_not_finite(backend_lib, dtype, V, copies, tail):
    from see_ml_b200 import token_ops as ops
    rng = np.random.default_rng(V)
    x = rng.standard_normal((8, V))
    ids, v = _teacher(rng, 8, V - 4, 6, F32)                   # the last four tokens are unnamed
    i = ids.cpu().numpy()
    low = float(torch.finfo(dtype).min)
    x[0, V - 1] = np.nan
    x[1, i[1, 2]] = np.nan
    x[2, V - 2] = np.inf
    x[3, i[3, 5]] = np.inf
    x[4] = -np.inf
    x[5] = low
    x[6, V - 4:] = low
    x[7, ::2] = -np.inf
    x[7, i[7]] = 1.0
    t = torch.from_numpy(x).to(dtype).cuda()
    loss, lerr, grad, gerr = R.distill(_f64(t)[4:], i[4:], _f64(v)[4:], 1.0, tail)
    many = t.repeat(copies, 1), ids.repeat(copies, 1), v.repeat(copies, 1)
    r = ops.distill_topk(*many, tail=tail, grad=True, saved=True)
    alone = ops.distill_topk(*many, tail=tail)
    g = ops.distill_topk_backward(*many, r.saved, torch.ones(8 * copies, device="cuda"), tail=tail)
    for c in {0, copies // 2, copies - 1}:
        mine = slice(8 * c, 8 * c + 8)
        for got in (r.row_loss[mine], alone.row_loss[mine]):
            assert got[:4].isnan().all()
            _close(got[4:], loss, lerr, F32, "row_loss")
        for got in (r.dlogits[mine], g[mine]):
            assert got[:4].isnan().all()
            _close(got[4:], grad, gerr, dtype, "dlogits")
