"""The fit operators on the GPU at their ends: empty and malformed inputs, the
forms and paths that ordinary sizes do not reach, and their torch ops."""

from __future__ import annotations

import importlib

import pytest
import torch

from golden_io import mb
from test_gpu_fit_ops import _bounds, _case

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops, _lib = mb.ops, mb._lib
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _stale(n, dtype):
    """Leaves NaN in the block that the next allocation of this size gets."""
    x = torch.full((n,), float("nan"), dtype=dtype, device=DEV)
    torch.cuda.synchronize()
    del x


# ------------------------------------------------------------- log probs
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 37, 5000])
def test_log_probs_gradient_without_segments(dtype, n):
    """Every element is outside every segment: its gradient is zero."""
    x = torch.randn(n, device=DEV).to(DT[dtype])
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    got = ops.log_probs(x, off)
    _stale(n + 8, x.dtype)
    dx = ops.log_probs_backward(x, off, None, got, torch.zeros(0, device=DEV))
    assert dx.shape == x.shape and torch.count_nonzero(dx) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,offsets,well", [
    (133, (0, 200, 133), ()), (133, (-5, 40, 133), (1,)), (133, (0, 50, 140), (0,)), (133, (0, 50, -3, 133), (0,)),
    (133, (150, 133, 133), ()), (70001, (0, 70002), ()), (70001, (0, 70002, 65000, 70001), (2,))])
def test_log_probs_gradient_of_malformed_segments(dtype, n, offsets, well):
    """A malformed segment is an error, and its elements have no gradient; the
    others' are what they are without it."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g).to(DT[dtype]).to(DEV)
    off = torch.tensor(offsets, device=DEV)
    p = off.shape[0] - 1
    gl, ge, gt = (torch.randn(*s, generator=g).to(DEV) for s in ((p,), (p,), (p, 3)))
    got = ops.log_probs(x, off, torch.zeros(p, dtype=torch.int64, device=DEV) - 1, top=3)
    with pytest.raises(ValueError, match="malformed"):
        mb._lib.check_device_error()
    _stale(n + 8, x.dtype)
    dx = ops.log_probs_backward(x, off, None, got, gl, ge, gt)
    with pytest.raises(ValueError, match="malformed"):
        mb._lib.check_device_error()
    want = torch.zeros_like(dx)
    for s in well:
        a, b = offsets[s], offsets[s + 1]
        one = torch.tensor([0, b - a], device=DEV)
        part = x[a:b].clone()
        alone = ops.log_probs(part, one, None, top=3)
        want[a:b] = ops.log_probs_backward(part, one, None, alone, gl[s:s + 1], ge[s:s + 1], gt[s:s + 1].contiguous())
    # the statistics' sums may be split otherwise: 2^-20 of terms of a few units, and a step of the type
    torch.testing.assert_close(dx.float(), want.float(), rtol=2.0 ** -7 if dtype == "bf16" else 2.0 ** -18, atol=2.0 ** -18)
    mb._lib.check_device_error()


# ------------------------------------------------------- the ops' autograd
torch_ops = importlib.import_module("hexo-shrimp-bot_b200.torch_ops")
torch_ops.define_fit()
fit = torch.ops.mantis_b200


def _attention_inputs(p, h, kv, length, d, dtype, seed=0, valid=None):
    """q, k, v (with gradients), bias, bucket map, coordinates, valid."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(p, n, length, d, generator=g).to(DT[dtype]).to(DEV).requires_grad_() for n in (h, kv, kv))
    bmap = torch.from_numpy(mb.hexgraph.displacement_buckets()).to(DEV)
    bias = torch.randn(int(bmap.max()) + 1, h, generator=g).to(DEV).requires_grad_()
    coords = torch.randint(-9, 10, (p, length, 2), generator=g, dtype=torch.int32).to(DEV)
    return q, k, v, bias, bmap, coords, valid


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("p,length", [(0, 5), (2, 0), (0, 0)])
def test_attention_autograd_of_an_empty_batch(dtype, p, length):
    args = _attention_inputs(p, 4, 2, length, 32, dtype)
    out = fit.bucket_attention(*args)[0]
    grads = torch.autograd.grad(out.float().sum(), args[:4])
    for x, y in zip(grads, args):
        assert x.shape == y.shape and x.dtype == y.dtype and torch.count_nonzero(x) == 0


def _segment_inputs(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(50, generator=g).to(DT[dtype]).to(DEV).requires_grad_()
    return x, torch.tensor([0, 20, 50], device=DEV), torch.tensor([3, 29], device=DEV), 2


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_outputs_without_a_gradient_formula(dtype):
    """A loss on a log-sum-exp raises; outputs that a loss leaves out cost the
    backward pass no zeros (the unrounded output's would be 4 MiB here)."""
    args = _attention_inputs(2, 4, 2, 4096, 32, dtype)
    out, lse, full = fit.bucket_attention(*args)
    seg = _segment_inputs(dtype)
    logp, entropy, seg_lse, top, top_logp = fit.log_probs(*seg)
    for aux in (lse, full, seg_lse):
        assert not aux.requires_grad
        with pytest.raises(RuntimeError, match="does not require grad"):
            aux.sum().backward()
    (dx,) = torch.autograd.grad(entropy.sum(), seg[0], retain_graph=True)
    want = ops.log_probs_backward(seg[0].detach(), *seg[1:3], ops.log_probs(*seg[:3], top=2), None,
                                  torch.ones(2, device=DEV))
    assert torch.equal(dx, want)
    go = torch.randn_like(out)
    stats = ops.AttentionStats(lse, full if dtype == "bf16" else None)
    peaks = []
    for run in (lambda: ops.bucket_attention_backward(*args, out.detach(), stats, go),
                lambda: torch.autograd.grad(out, args[:4], go)):
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with torch.no_grad():
            run()
        peaks.append(torch.cuda.max_memory_allocated() - before)
    assert peaks[1] <= peaks[0] + (1 << 20)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_compiled_step(dtype):
    """A traced fit step (forward and backward, no break in the graph) gives
    the eager step's loss and gradients bit for bit, over steps whose dropout
    seed changes, and is traced twice at most (the second time with the seed
    as a symbol)."""
    from torch._dynamo.testing import CompileCounterWithBackend

    torch._dynamo.reset()
    torch.manual_seed(3)
    cfg = mb.policy.PolicyConfig(h=64, blocks=2, heads=2, kv_heads=1, dropout=0.2)
    model = mb.policy.CellPolicy(cfg, dtype=DT[dtype]).cuda()
    batch = mb.policy.token_batch(mb.engine.random_positions(3, 4, 12, seed=5))
    played = (batch.kind == mb.policy.EMPTY).long().argmax(1)
    counter = CompileCounterWithBackend("aot_eager")
    step = torch.compile(lambda seed: model.loss(batch, played, 0.05, seed=seed), backend=counter, fullgraph=True)
    for seed in (11, 12, 13, 14):
        results = []
        for run in (lambda: model.loss(batch, played, 0.05, seed=seed), lambda: step(seed)):
            model.zero_grad(set_to_none=True)
            loss = run()
            loss.backward()
            results.append([loss.detach(), *(t.grad for t in model.parameters() if t is not model.embed.weight)])
        for x, y in zip(*results):
            assert torch.equal(x, y)
    assert counter.frame_count <= 2
    mb._lib.check_device_error()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_second_derivatives(dtype):
    """First gradients are the same with and without create_graph. Through
    attention and log probabilities a second one raises; dropout's, of a
    function quadratic in y, is the mask and gain twice."""
    args = _attention_inputs(1, 2, 1, 9, 32, dtype)
    seg = _segment_inputs(dtype)
    for run, xs in ((lambda: fit.bucket_attention(*args)[0].float().sum(), args[:4]),
                    (lambda: fit.log_probs(*seg)[0].sum(), seg[:1]),
                    (lambda: fit.log_probs(*seg)[1].square().sum(), seg[:1])):
        plain = torch.autograd.grad(run(), xs)
        grads = torch.autograd.grad(run(), xs, create_graph=True)
        assert all(torch.equal(a, b) and b.requires_grad for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(sum(x.float().square().sum() for x in grads), xs[0])
        loss = run() + 0.1 * sum(x.float().square().sum() for x in grads)  # a penalty beside a loss
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(loss, xs[0])
    x = torch.randn(6, 40, device=DEV)
    y = torch.randn(6, 40, device=DEV).to(DT[dtype]).requires_grad_()
    out = fit.dropout_add(x, y, 0.5, 7, 3)
    (dy,) = torch.autograd.grad((0.5 * (out - x).square()).sum(), y, create_graph=True)
    (ddy,) = torch.autograd.grad(dy.float().sum(), y)
    keep = (out.detach() != x).to(ddy.dtype)
    assert torch.equal(ddy, 4 * keep)  # a gain of 2, twice: exact


def test_log_probs_outputs_share_no_memory():
    """An in-place step on one output leaves the others and the gradient right."""
    x, off, ranks, top = _segment_inputs("f32")
    logp, entropy, lse, *_ = fit.log_probs(x, off, ranks, top)
    assert len({t.untyped_storage().data_ptr() for t in (logp, entropy, lse)}) == 3
    kept = entropy.detach().clone(), lse.clone()
    (want,) = torch.autograd.grad(3 * logp.sum(), x, retain_graph=True)
    logp *= 3
    (got,) = torch.autograd.grad(logp.sum(), x)
    assert torch.equal(got, want) and torch.equal(entropy, kept[0]) and torch.equal(lse, kept[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ops_keep_the_custom_op_contract(dtype):
    """Schemas (no mutation, no aliasing), autograd keys and fakes, by torch's own check."""
    which = ("test_schema", "test_autograd_registration", "test_faketensor")
    args = _attention_inputs(2, 4, 2, 9, 32, dtype, valid=torch.tensor([9, 4], dtype=torch.int32, device=DEV))
    seg = _segment_inputs(dtype)
    y = torch.randn(3, 8, device=DEV).to(DT[dtype])
    out, lse, full = (t.detach() for t in fit.bucket_attention(*args))
    logp, entropy, seg_lse, tops, top_logp = (t.detach() for t in fit.log_probs(*seg))
    flat = [t.detach() for t in args]
    for op, a in ((fit.bucket_attention, args), (fit.log_probs, seg),
                  (fit.dropout_add, (y.float().requires_grad_(), y.clone().requires_grad_(), 0.3, 5, 6)),
                  (fit.bucket_attention_backward, (*flat, out, lse, full, out, None, True)),
                  (fit.log_probs_backward, (seg[0].detach(), *seg[1:3], seg_lse, entropy, tops, logp, entropy, top_logp)),
                  (fit.dropout_backward, (y, 0.3, 5, 6, torch.float32))):
        torch.library.opcheck(op.default, a, test_utils=which)


def test_log_probs_backward_refuses_another_result():
    """A result on the host, of another type or of other segments is refused
    before any launch."""
    x, off, ranks, top = _segment_inputs("f32")
    x = x.detach()
    got = ops.log_probs(x, off, ranks, top=top)
    g = torch.ones(2, device=DEV)
    short = ops.log_probs(x, off[:2], ranks[:1], top=top)
    wide = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    for bad in (got._replace(lse=got.lse.cpu()), got._replace(entropy=got.entropy.cpu()),
                got._replace(top=got.top.cpu()), got._replace(lse=got.lse.double()),
                got._replace(entropy=got.entropy.bfloat16()), got._replace(entropy=short.entropy),
                got._replace(top=got.top.int()), got._replace(top=short.top), got._replace(top=got.top[:, 0]),
                got._replace(top=wide[:, ::2]), got._replace(top=torch.zeros(2, 33, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError, match="result of log_probs"):
            ops.log_probs_backward(x, off, ranks, bad, g)
    with pytest.raises(ValueError, match="g_top"):
        ops.log_probs_backward(x, off, ranks, got, g, None, torch.ones(2, 3, device=DEV))


# ------------------------------------------------- attention's other forms
def _to_device(args):
    """q, k, v as views of one fused tensor, then go and the rest, on the device."""
    q, k, v, go, *rest = args
    fused = torch.cat([q, k, v], 1).permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
    return (*fused.split([q.shape[1], k.shape[1], k.shape[1]], 1), go.to(DEV),
            *(x.to(DEV) if x is not None else None for x in rest))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("length,layout,ragged", [(1, "hex", False), (37, "hex", False), (129, "causal", True),
                                                  (200, "hex", True), (257, "line", True), (513, "line", False),
                                                  (1100, "line", False)])
def test_attention_serving_form(dtype, d, length, layout, ragged):
    """The form that keeps nothing for a backward pass, elementwise against the
    oracle: its bound has the probabilities' and the output's roundings to
    bf16, and no more."""
    args = _case(1 if length > 500 else 3, 4, 2, length, d, dtype, layout, ragged=ragged, seed=130)
    (want, want_lse, *_), (bound, bound_lse, *_) = _bounds(*args, dtype)
    q, k, v, _, *rest = _to_device(args)
    out, lse = ops.bucket_attention(q, k, v, *rest, with_lse=True)
    for name, x, y, b in (("out", out, want, bound), ("lse", lse, want_lse, bound_lse)):
        x = x.double().cpu()
        fin = torch.isfinite(y)
        assert torch.equal(fin, torch.isfinite(x)) and torch.equal(x[~fin], y[~fin]), name
        over = ((x - y).abs() - b)[fin]
        assert over.numel() == 0 or float(over.max()) <= 1e-12, f"{name}: {float(over.max()):.3e} over its bound"
    mb._lib.check_device_error()


def _within(name, got, want, bound):
    got = got.detach().double().cpu()
    over = (got - want).abs() - bound
    assert got.shape == want.shape
    assert over.numel() == 0 or float(over.max()) <= 1e-12, f"{name}: {float(over.max()):.3e} over its bound"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bias_grad", [True, False])
@pytest.mark.parametrize("heads,kv,length,d", [(4, 4, 70, 32), (4, 1, 140, 64)])
def test_attention_autograd_matches_the_oracle(dtype, bias_grad, heads, kv, length, d):
    """The torch op's gradients, from strided views and a gradient in another layout."""
    args = _case(3, heads, kv, length, d, dtype, ragged=True, seed=131)
    want, bound = _bounds(*args, dtype)
    q, k, v, go, bias, *rest = _to_device(args)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + [bias.requires_grad_(bias_grad)]
    out, lse, _ = fit.bucket_attention(*leaves, *rest)
    grads = torch.autograd.grad(out, leaves if bias_grad else leaves[:3], go)
    for name, x, y, b in zip(("out", "dq", "dk", "dv", "dbias"), (out, *grads), (want[0], *want[2:]),
                             (bound[0], *bound[2:])):
        _within(name, x, y, b)
    mb._lib.check_device_error()


@pytest.mark.parametrize("d,heads,kv", [(32, 2, 2), (64, 4, 1), (128, 2, 1)])
@pytest.mark.parametrize("parts", [1, 2, 4, 5, 6])
def test_attention_gradients_in_chunks_of_key_tiles(d, heads, kv, parts):
    """Six key tiles, `parts` of dQ kept at a time: the running sum over
    chunks, a last chunk of fewer tiles, and positions that end in the first
    chunk, against the oracle; the same again bit for bit."""
    length = 700
    args = list(_case(3, heads, kv, length, d, "bf16", "line", seed=140))
    args[-1] = torch.tensor([700, 130, 391], dtype=torch.int32)
    want, bound = _bounds(*args, "bf16")
    q, k, v, go, *rest = _to_device(args)
    try:
        ops.bucket_attention_limit_parts(parts * 4 * 3 * heads * length * d)
        out, st = ops.bucket_attention(q, k, v, *rest, for_backward=True)
        grads = ops.bucket_attention_backward(q, k, v, *rest, out, st, go)
        again = ops.bucket_attention_backward(q, k, v, *rest, out, st, go)
    finally:
        ops.bucket_attention_limit_parts(0)
    for name, x, x2, y, b in zip(("dq", "dk", "dv", "dbias"), grads, again, want[2:], bound[2:]):
        _within(name, x, y, b)
        assert torch.equal(x, x2)
    mb._lib.check_device_error()


@pytest.mark.parametrize("dtype,d,p,length", [("bf16", 32, 3, 300), ("bf16", 64, 40, 70), ("bf16", 16, 3, 150),
                                              ("f32", 32, 3, 150)])
def test_attention_gradients_within_their_workspace(dtype, d, p, length):
    """Through the C entry with the workspace that it asks for and not a byte
    more, on rows of 16 bytes and off them (the CUDA cores, with the bias sums
    where the tensor cores keep their parts): the same gradients as the wrapper's
    to the roundings between the two paths, and the bytes behind it untouched."""
    args = _case(p, 4, 2, length, d, dtype, ragged=True, seed=150)
    want, bound = _bounds(*args, dtype)
    q, k, v, go, bias, bmap, coords, valid = _to_device(args)
    wide = [torch.empty(*t.shape[:3], d + 1, dtype=t.dtype, device=DEV)[..., 1:] for t in (q, k, v)]
    for w, t in zip(wide, (q, k, v)):
        w.copy_(t)
    for q, k, v in ((q, k, v), wide):
        out, st = ops.bucket_attention(q, k, v, bias, bmap, coords, valid, for_backward=True)
        kept, fixed = ops._bucket_args(q, k, v, bias, bmap, coords, valid, None)
        need = ops._bucket_workspace(_lib.dtype_code(q.dtype), p, 4, 2, d, length, bias.shape[0])
        ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in (q, k, v))
        dbias = torch.empty_like(bias)
        g = go.contiguous()
        _lib.call("mb_bucket_attention_backward", *fixed, out.data_ptr(), *out.stride()[:3], _lib.ptr(st.full),
                  st.lse.data_ptr(), g.data_ptr(), *g.stride()[:3], ws.data_ptr(), need, dq.data_ptr(), dk.data_ptr(),
                  dv.data_ptr(), dbias.data_ptr(), _lib.stream_of(q.device))
        for name, x, y, b in zip(("dq", "dk", "dv", "dbias"), (dq, dk, dv, dbias), want[2:], bound[2:]):
            _within(name, x, y, b)
        assert bool((ws[need:] == 0xA5).all())
    mb._lib.check_device_error()


def test_attention_gradients_of_unaligned_rows_reserve_no_parts():
    """bf16 rows off 16 bytes run on the CUDA cores: beside the gradients they
    need delta and the bias sums (4 MiB here), not the 1 GiB of dQ's parts that
    the same rows on 16 bytes keep, and the results agree."""
    p, h, length, d = 64, 8, 1024, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = [torch.randn(p, h, length, d + 1, generator=g, device=DEV).bfloat16() for _ in range(3)]
    bmap = torch.from_numpy(mb.hexgraph.line_buckets()).to(DEV)
    bias = torch.randn(32, h, generator=g, device=DEV)
    t = torch.arange(length, dtype=torch.int32, device=DEV)
    where = bias, bmap, torch.stack([t, torch.zeros_like(t)], -1).contiguous(), None
    results, extra = [], []
    for q, k, v in ([r[..., 1:] for r in rows], [r[..., 1:].contiguous() for r in rows]):
        out, st = ops.bucket_attention(q, k, v, *where, for_backward=True)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        grads = ops.bucket_attention_backward(q, k, v, *where, out, st, out)
        extra.append(torch.cuda.max_memory_allocated() - before - sum(x.numel() * x.element_size() for x in grads))
        results.append(grads)
    assert extra[0] <= 8 << 20 and extra[1] >= 1 << 30
    # P and dS are rounded to bf16 on the tensor cores alone: 2^-9 of terms, 2^-7 of the largest sum
    for x, y in zip(*results):
        assert float((x.float() - y.float()).abs().max()) <= 2.0 ** -7 * float(y.float().abs().max())
    mb._lib.check_device_error()
