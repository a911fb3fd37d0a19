"""The operator-level plug-in: this library's kernels behind the reference's
``mantisnet::`` torch.library custom ops.

The reference registers each data-dependent forward of MantisNet as an
opaque custom op (e.g. python/mantisnet/mantisnet/attention.py:719-753,
cell_latents.py:834-860, window_latents.py:553-714, message_passing.py:191-365,
row_encoder.py:368-380, relay.py:452) with a ``register_fake`` so that
``torch.compile(dynamic=True, fullgraph=True)`` keeps it opaque. Two ways in:

- :func:`install_into_reference` registers a CUDA kernel of this library for
  every one of those ops that is already defined (the reference package
  imported), so the reference's own ``MantisNet`` runs its op calls on these
  kernels; the reference's fakes and CPU paths stay as they are.
- :func:`define` defines the same ops (names, argument lists, output
  contracts) in a namespace of their own (default ``mantis_b200``) with these
  kernels and fake implementations, for callers without the reference.

Backward: :func:`define` registers autograd for the attention ops and the
action-row encoder on this library's deterministic backward kernels, and
:func:`install_into_reference` also takes over the reference's backward ops
(``*_backward``, e.g. attention.py:823-890, cell_latents.py:869-990,
window_latents.py:589-700), so the reference's own autograd formulas call
these kernels. Every output follows the reference op's contract, auxiliary
statistics included (fused_attention's per-row log-sum-exp, the segment
attentions' running max and sum).

:func:`define_fit` defines the fit operators, which the reference does not
have (bucketed relative-bias attention, dropout on a residual branch, log
probabilities of chosen moves), with fakes and autograd.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor

from . import ops

# op name -> schema (the reference's argument names and types)
_SCHEMAS = {
    "fused_attention": "(Tensor q, Tensor k, Tensor v, Tensor seq_lens) -> (Tensor, Tensor)",
    "cell_attention": ("(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor vcls, Tensor seg_ptr, Tensor src, "
                       "Tensor cls, Tensor qid, Tensor sseg_ptr, Tensor sqid, Tensor scls, Tensor cptr, "
                       "Tensor cedge_q) -> (Tensor, Tensor, Tensor)"),
    "cell_attention_plain": ("(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor seg_ptr, Tensor src, Tensor cls, "
                             "Tensor qid, Tensor sseg_ptr, Tensor sqid, Tensor scls, Tensor cptr, Tensor cedge_q) "
                             "-> (Tensor, Tensor, Tensor)"),
    "window_latent_read": ("(Tensor q, Tensor k, Tensor v, Tensor window_pos, Tensor offsets, Tensor order) "
                           "-> (Tensor, Tensor, Tensor)"),
    "window_latent_broadcast": ("(Tensor q, Tensor k, Tensor v, Tensor window_pos, Tensor offsets, Tensor order) "
                                "-> (Tensor, Tensor, Tensor)"),
    "aggregate_to_windows": ("(Tensor values, Tensor inc_stone, Tensor inc_window, Tensor run_stone, "
                             "Tensor run_window, int n_windows) -> Tensor"),
    "aggregate_to_stones": ("(Tensor values, Tensor inc_stone, Tensor inc_window, Tensor run_stone, "
                            "Tensor run_window, int n_stones) -> Tensor"),
    "class_row_sum": "(Tensor weight, Tensor gather, Tensor runs, int n_dest, int run_len) -> Tensor",
    "incidence_row_sum": ("(Tensor values, Tensor gather, Tensor runs, Tensor rev_gather, Tensor rev_runs, "
                          "int n_dest, int run_len, int rev_run_len) -> Tensor"),
    "action_row_encode": ("(Tensor pre_w, Tensor table, Tensor edge_window, Tensor edge_class, Tensor edge_cell, "
                          "Tensor edge_rev, int n_cells) -> Tensor"),
    "cell_pass": ("(Tensor x, Tensor emb, Tensor cell_ptr, Tensor edge_window, Tensor edge_class, Tensor win_ptr, "
                  "Tensor edge_wcell, Tensor cls_ptr, Tensor edge_ccell) -> Tensor"),
    "window_latent_layout": "(Tensor window_pos, int positions) -> (Tensor, Tensor)",
}


def _lse_wanted(q: Tensor) -> bool:
    """The reference returns a (P, A, T) log-sum-exp when its CUDA kernel
    serves the shape (fp16 / bf16, head_dim 16, 32 or 64), else an empty one
    (attention.py:727-732, 756-772)."""
    return q.is_cuda and q.dtype in (torch.float16, torch.bfloat16) and q.shape[-1] in (16, 32, 64)


# ------------------------------------------------------------ CUDA kernels
def _fused_attention(q, k, v, seq_lens):
    if q.dtype == torch.float16:
        raise NotImplementedError("mantisnet::fused_attention on this library takes bf16 or fp32 tensors")
    if _lse_wanted(q):
        return ops.fused_attention(q, k, v, seq_lens, with_lse=True)
    return ops.fused_attention(q, k, v, seq_lens), torch.empty(0, dtype=torch.float32, device=q.device)


def _cell_attention(q, k, v, bias, vcls, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q):
    return tuple(ops.cell_attention(q, k, v, bias, vcls, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q))


def _cell_attention_plain(q, k, v, bias, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q):
    return tuple(ops.cell_attention_plain(q, k, v, bias, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q))


def _window_latent_read(q, k, v, window_pos, offsets, order):
    p, _, heads, hd = q.shape
    out, m, l = ops.latent_read(q.reshape(p * 4, -1).contiguous(), k.reshape(k.shape[0], -1).contiguous(),
                                v.reshape(v.shape[0], -1).contiguous(), heads, offsets, order, stats=True)
    return out.view(q.shape), m.view(q.shape[:-1]), l.view(q.shape[:-1])


def _window_latent_broadcast(q, k, v, window_pos, offsets, order):
    n_w, heads, hd = q.shape
    out, m, l = ops.latent_broadcast(q.reshape(n_w, -1).contiguous(), k.reshape(-1, heads * hd).contiguous(),
                                     v.reshape(-1, heads * hd).contiguous(), heads, window_pos, k.shape[0],
                                     stats=True)
    return out.view(q.shape), m.view(q.shape[:-1]), l.view(q.shape[:-1])


def _window_latent_layout(window_pos, positions):
    return tuple(ops.window_latent_layout(window_pos, positions))


_KERNELS = {
    "fused_attention": _fused_attention,
    "cell_attention": _cell_attention,
    "cell_attention_plain": _cell_attention_plain,
    "window_latent_read": _window_latent_read,
    "window_latent_broadcast": _window_latent_broadcast,
    "aggregate_to_windows": ops.aggregate_to_windows,
    "aggregate_to_stones": ops.aggregate_to_stones,
    "class_row_sum": ops.class_row_sum,
    "incidence_row_sum": ops.incidence_row_sum,
    "action_row_encode": ops.encode_rows,
    "cell_pass": ops.cell_pass,
    "window_latent_layout": _window_latent_layout,
}


# ------------------------------------------------------------- fakes
def _fake_fused_attention(q, k, v, seq_lens):
    lse = (q.new_empty(q.shape[:3], dtype=torch.float32) if _lse_wanted(q)
           else q.new_empty((0,), dtype=torch.float32))
    return torch.empty_like(q), lse


def _fake_segment(q, *rest):
    n_q, heads, hd = q.shape
    return (q.new_empty((n_q, heads, hd), dtype=torch.float32), q.new_empty((n_q, heads), dtype=torch.float32),
            q.new_empty((n_q, heads), dtype=torch.float32))


def _fake_latent(q, k, v, window_pos, offsets, order):
    return (q.new_empty(q.shape, dtype=torch.float32), q.new_empty(q.shape[:-1], dtype=torch.float32),
            q.new_empty(q.shape[:-1], dtype=torch.float32))


def _fake_aggregate_to_windows(values, inc_stone, inc_window, run_stone, run_window, n_windows):
    return values.new_empty((n_windows, values.shape[1]))


def _fake_aggregate_to_stones(values, inc_stone, inc_window, run_stone, run_window, n_stones):
    return values.new_empty((n_stones, values.shape[1]), dtype=torch.float32)


def _fake_class_row_sum(weight, gather, runs, n_dest, run_len):
    return weight.new_empty((n_dest, weight.shape[1]), dtype=torch.float32)


def _fake_incidence_row_sum(values, gather, runs, rev_gather, rev_runs, n_dest, run_len, rev_run_len):
    return values.new_empty((n_dest, values.shape[1]), dtype=torch.float32)


def _fake_action_row_encode(pre_w, table, edge_window, edge_class, edge_cell, edge_rev, n_cells):
    return pre_w.new_empty((n_cells, pre_w.shape[1]), dtype=torch.float32)


def _fake_cell_pass(x, emb, cell_ptr, edge_window, edge_class, win_ptr, edge_wcell, cls_ptr, edge_ccell):
    return torch.empty_like(x)


def _fake_window_latent_layout(window_pos, positions):
    return window_pos.new_empty((positions + 1,), dtype=torch.long), torch.empty_like(window_pos)


_FAKES = {
    "fused_attention": _fake_fused_attention,
    "cell_attention": _fake_segment,
    "cell_attention_plain": _fake_segment,
    "window_latent_read": _fake_latent,
    "window_latent_broadcast": _fake_latent,
    "aggregate_to_windows": _fake_aggregate_to_windows,
    "aggregate_to_stones": _fake_aggregate_to_stones,
    "class_row_sum": _fake_class_row_sum,
    "incidence_row_sum": _fake_incidence_row_sum,
    "action_row_encode": _fake_action_row_encode,
    "cell_pass": _fake_cell_pass,
    "window_latent_layout": _fake_window_latent_layout,
}

_libs: dict[str, torch.library.Library] = {}


def define(namespace: str = "mantis_b200") -> list[str]:
    """Define every op of the plug-in in ``namespace`` (reference names,
    argument lists and output contracts) with this library's CUDA kernels
    and fake implementations. Returns the qualified op names. Idempotent."""
    names = [f"{namespace}::{n}" for n in _SCHEMAS]
    if namespace in _libs:
        return names
    lib = torch.library.Library(namespace, "FRAGMENT")
    for name, schema in _SCHEMAS.items():
        lib.define(name + schema)
        lib.impl(name, _KERNELS[name], "CUDA")
        torch.library.register_fake(f"{namespace}::{name}", _FAKES[name], lib=lib)
        if name in _AUTOGRAD:
            torch.library.register_autograd(f"{namespace}::{name}", _AUTOGRAD[name], setup_context=_save_all,
                                            lib=lib)
    _libs[namespace] = lib
    return names


def install_into_reference(namespace: str = "mantisnet") -> list[str]:
    """Register this library's kernels as the CUDA implementation of each of
    the reference's ops that is defined (import the reference package
    first). Returns the ops it took over."""
    taken = []
    for name, fn in list(_KERNELS.items()) + list(_BACKWARD_KERNELS.items()):
        qual = f"{namespace}::{name}"
        try:
            torch._C._dispatch_find_schema_or_throw(qual, "")
        except RuntimeError:
            continue
        torch.library.register_kernel(qual, "cuda", fn)
        taken.append(qual)
    return taken


# ------------------------------------------------------------ backward
# The reference's backward ops (same argument lists), on this library's
# deterministic backward kernels.
def _fused_attention_backward(q, k, v, seq_lens, out, lse, grad_out):
    if lse.numel() == 0:  # a forward that kept no log-sum-exp: recompute it
        _, lse = ops.fused_attention(q, k, v, seq_lens, with_lse=True)
    return ops.stone_attention_backward(q, k, v, seq_lens, out, lse, grad_out)


def _cell_attention_backward(q, k, v, bias, vcls, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q, m,
                             l, grad_out):
    return ops.segment_attention_backward(q, k, v, bias, vcls, seg_ptr, src, cls, m, l, grad_out, qid=qid)


def _cell_attention_plain_backward(q, k, v, bias, seg_ptr, src, cls, qid, sseg_ptr, sqid, scls, cptr, cedge_q, m,
                                   l, grad_out):
    return ops.segment_attention_backward(q, k, v, bias, None, seg_ptr, src, cls, m, l, grad_out, qid=qid)[:4]


def _window_latent_read_backward(q, k, v, window_pos, offsets, order, out, m, l, grad_out):
    return ops.window_latent_read_backward(q, k, v, offsets, order, window_pos, out, m, l, grad_out)


def _window_latent_broadcast_backward(q, k, v, window_pos, offsets, order, m, l, grad_out):
    return ops.window_latent_broadcast_backward(q, k, v, offsets, order, window_pos, m, l, grad_out)


_BACKWARD_KERNELS = {
    "fused_attention_backward": _fused_attention_backward,
    "cell_attention_backward": _cell_attention_backward,
    "cell_attention_plain_backward": _cell_attention_plain_backward,
    "window_latent_read_backward": _window_latent_read_backward,
    "window_latent_broadcast_backward": _window_latent_broadcast_backward,
}


# Autograd of the ops :func:`define` creates: save what the backward reads,
# return one gradient per input (None for index tensors and ints).
def _save_all(ctx, inputs, output):
    outs = output if isinstance(output, tuple) else (output,)
    ctx.save_for_backward(*[x for x in inputs if isinstance(x, torch.Tensor)],
                          *[o for o in outs if isinstance(o, torch.Tensor)])
    ctx.n_in = sum(isinstance(x, torch.Tensor) for x in inputs)
    ctx.ints = [x for x in inputs if not isinstance(x, torch.Tensor)]


def _bw_fused_attention(ctx, g_out, g_lse):
    q, k, v, seq_lens, out, lse = ctx.saved_tensors
    return (*_fused_attention_backward(q, k, v, seq_lens, out, lse, g_out), None)


def _bw_cell_attention(ctx, g_out, g_m, g_l):
    t = ctx.saved_tensors
    q, k, v, bias, vcls, seg_ptr, src, cls, qid = t[:9]
    m, l = t[15], t[16]
    return (*ops.segment_attention_backward(q, k, v, bias, vcls, seg_ptr, src, cls, m, l, g_out, qid=qid),
            *([None] * 9))


def _bw_cell_attention_plain(ctx, g_out, g_m, g_l):
    t = ctx.saved_tensors
    q, k, v, bias, seg_ptr, src, cls, qid = t[:8]
    m, l = t[14], t[15]
    return (*ops.segment_attention_backward(q, k, v, bias, None, seg_ptr, src, cls, m, l, g_out, qid=qid)[:4],
            *([None] * 9))


def _bw_window_latent_read(ctx, g_out, g_m, g_l):
    q, k, v, window_pos, offsets, order, out, m, l = ctx.saved_tensors
    return (*ops.window_latent_read_backward(q, k, v, offsets, order, window_pos, out, m, l, g_out), None, None,
            None)


def _bw_window_latent_broadcast(ctx, g_out, g_m, g_l):
    q, k, v, window_pos, offsets, order, out, m, l = ctx.saved_tensors
    return (*ops.window_latent_broadcast_backward(q, k, v, offsets, order, window_pos, m, l, g_out), None, None,
            None)


def _bw_action_row_encode(ctx, g_out):
    pre_w, table, edge_window, edge_class, edge_cell, edge_rev, out = ctx.saved_tensors
    gp, gt = ops.encode_rows_backward(pre_w, table, edge_window, edge_class, edge_cell, g_out)
    return gp, gt, None, None, None, None, None


_AUTOGRAD = {
    "fused_attention": _bw_fused_attention,
    "cell_attention": _bw_cell_attention,
    "cell_attention_plain": _bw_cell_attention_plain,
    "window_latent_read": _bw_window_latent_read,
    "window_latent_broadcast": _bw_window_latent_broadcast,
    "action_row_encode": _bw_action_row_encode,
}


# ------------------------------------------------------------ fit operators
# Each differentiable op, and the op that its backward formula calls: an op of
# its own, so that a traced backward pass keeps it opaque too. Seeds and
# offsets are symbolic: they change every step, and a compiled one stays.
_FIT_SCHEMAS = {
    "bucket_attention": ("(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor bucket_map, Tensor coords, "
                         "Tensor? valid, float? scale=None) -> (Tensor, Tensor, Tensor)"),
    "dropout_add": "(Tensor x, Tensor y, float p, SymInt seed, SymInt offset) -> Tensor",
    "log_probs": ("(Tensor logits, Tensor offsets, Tensor ranks, int top=0) "
                  "-> (Tensor, Tensor, Tensor, Tensor, Tensor)"),
}
_FIT_BACKWARD_SCHEMAS = {
    "bucket_attention_backward": ("(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor bucket_map, Tensor coords, "
                                  "Tensor? valid, Tensor out, Tensor lse, Tensor full, Tensor grad_out, "
                                  "float? scale=None, bool bias_grad=True) -> (Tensor, Tensor, Tensor, Tensor)"),
    "dropout_backward": "(Tensor grad, float p, SymInt seed, SymInt offset, ScalarType dtype) -> Tensor",
    "log_probs_backward": ("(Tensor logits, Tensor offsets, Tensor ranks, Tensor lse, Tensor entropy, Tensor top, "
                           "Tensor? g_logp, Tensor? g_entropy, Tensor? g_top_logp) -> Tensor"),
}


def _fit_bucket_attention(q, k, v, bias, bucket_map, coords, valid, scale=None):
    out, stats = ops.bucket_attention(q, k, v, bias, bucket_map, coords, valid, scale=scale, for_backward=True)
    full = stats.full if stats.full is not None else torch.empty(0, dtype=torch.float32, device=q.device)
    return out, stats.lse, full


def _fit_bucket_attention_backward(q, k, v, bias, bucket_map, coords, valid, out, lse, full, grad_out, scale=None,
                                   bias_grad=True):
    stats = ops.AttentionStats(lse, full if q.dtype == torch.bfloat16 else None)
    dq, dk, dv, dbias = ops.bucket_attention_backward(q, k, v, bias, bucket_map, coords, valid, out, stats, grad_out,
                                                      scale=scale, bias_grad=bias_grad)
    return dq, dk, dv, bias.new_empty(0) if dbias is None else dbias


def _fit_log_probs(logits, offsets, ranks, top=0):
    return tuple(ops.log_probs(logits, offsets, ranks, top=top))


def _fit_log_probs_backward(logits, offsets, ranks, lse, entropy, top, g_logp, g_entropy, g_top_logp):
    got = ops.LogProbs(None, entropy, lse, top, None)  # what the kernel reads
    return ops.log_probs_backward(logits, offsets, ranks, got, g_logp, g_entropy, g_top_logp)


_FIT_KERNELS = {"bucket_attention": _fit_bucket_attention, "dropout_add": ops.dropout_add,
                "log_probs": _fit_log_probs, "bucket_attention_backward": _fit_bucket_attention_backward,
                "dropout_backward": ops.dropout_backward, "log_probs_backward": _fit_log_probs_backward}


def _fake_bucket_attention(q, k, v, bias, bucket_map, coords, valid, scale=None):
    full = q.shape if q.dtype == torch.bfloat16 else (0,)
    return (q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32),
            q.new_empty(full, dtype=torch.float32))


def _fake_bucket_attention_backward(q, k, v, bias, bucket_map, coords, valid, out, lse, full, grad_out, scale=None,
                                    bias_grad=True):
    return (q.new_empty(q.shape), k.new_empty(k.shape), k.new_empty(k.shape),
            bias.new_empty(bias.shape if bias_grad else 0))


def _fake_dropout_add(x, y, p, seed, offset):
    return x.new_empty(x.shape)


def _fake_dropout_backward(grad, p, seed, offset, dtype):
    return grad.new_empty(grad.shape, dtype=dtype)


def _fake_log_probs(logits, offsets, ranks, top=0):
    p = offsets.shape[0] - 1
    f = lambda *s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    return f(p), f(p), f(p), logits.new_empty((p, top), dtype=torch.long), f(p, top)


def _fake_log_probs_backward(logits, offsets, ranks, lse, entropy, top, g_logp, g_entropy, g_top_logp):
    return logits.new_empty(logits.shape)


_FIT_FAKES = {"bucket_attention": _fake_bucket_attention, "dropout_add": _fake_dropout_add,
              "log_probs": _fake_log_probs, "bucket_attention_backward": _fake_bucket_attention_backward,
              "dropout_backward": _fake_dropout_backward, "log_probs_backward": _fake_log_probs_backward}


# The backward formulas call the backward op of the forward op's namespace.
def _save_bucket_attention(ctx, inputs, output):
    q, k, v, bias, bucket_map, coords, valid, ctx.scale = inputs
    ctx.mark_non_differentiable(*output[1:])
    ctx.set_materialize_grads(False)  # the aux outputs' zeros would be as large as out's
    ctx.save_for_backward(q, k, v, bias, bucket_map, coords, valid, *output)


def _bw_bucket_attention(op, ctx, g_out, g_lse, g_full):
    if g_out is None:
        return (None,) * 8
    dq, dk, dv, dbias = op(*ctx.saved_tensors, g_out, ctx.scale, ctx.needs_input_grad[3])
    return dq, dk, dv, dbias if ctx.needs_input_grad[3] else None, None, None, None, None


def _save_dropout_add(ctx, inputs, output):
    _, y, ctx.p, ctx.seed, ctx.offset = inputs
    ctx.y_dtype = y.dtype


def _bw_dropout_add(op, ctx, g):
    return g, op(g, ctx.p, ctx.seed, ctx.offset, ctx.y_dtype), None, None, None


def _save_log_probs(ctx, inputs, output):
    ctx.mark_non_differentiable(*output[2:4])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*inputs[:3], output[2], output[1], output[3])


def _bw_log_probs(op, ctx, g_logp, g_entropy, g_lse, g_top, g_top_logp):
    grads = [None if g is None else g.float().contiguous() for g in (g_logp, g_entropy, g_top_logp)]
    if grads[2] is not None and grads[2].numel() == 0:
        grads[2] = None
    return op(*ctx.saved_tensors, *grads), None, None, None


# Second derivatives: dropout's gradient is linear in its argument, with the
# forward's mask; the others have no formula, and say so where one is asked
# for rather than stand as constants.
def _save_dropout_backward(ctx, inputs, output):
    grad, ctx.p, ctx.seed, ctx.offset, _ = inputs
    ctx.grad_dtype = grad.dtype


def _bw_dropout_backward(op, ctx, g):
    return op(g, ctx.p, ctx.seed, ctx.offset, ctx.grad_dtype), None, None, None, None


def _no_second(name):
    def backward(ctx, *grads):
        raise RuntimeError(f"{name} has no second derivative")
    return backward


_FIT_AUTOGRAD = {"bucket_attention": (_bw_bucket_attention, _save_bucket_attention),
                 "dropout_add": (_bw_dropout_add, _save_dropout_add),
                 "log_probs": (_bw_log_probs, _save_log_probs)}
_FIT_BACKWARD_OP = {"bucket_attention": "bucket_attention_backward", "dropout_add": "dropout_backward",
                    "log_probs": "log_probs_backward"}


def define_fit(namespace: str = "mantis_b200") -> list[str]:
    """Define the fit operators in ``namespace`` with this library's CUDA
    kernels, fakes and autograd; their backward passes are ops with fakes too, so
    a training step traces. Second derivatives: dropout has them, the other two
    raise where one is asked for. ``bucket_attention`` returns (out, lse, full):
    the log-sum-exp and the unrounded output are kept for the backward pass
    and are not differentiable (``requires_grad`` is False), nor is
    ``log_probs``'s lse (its logp, entropy and top_logp are). Returns the
    differentiable ops' qualified names. Idempotent."""
    names = [f"{namespace}::{n}" for n in _FIT_SCHEMAS]
    key = f"{namespace} (fit)"
    if key in _libs:
        return names
    lib = torch.library.Library(namespace, "FRAGMENT")
    for name, schema in {**_FIT_SCHEMAS, **_FIT_BACKWARD_SCHEMAS}.items():
        lib.define(name + schema)
        lib.impl(name, _FIT_KERNELS[name], "CUDA")
        torch.library.register_fake(f"{namespace}::{name}", _FIT_FAKES[name], lib=lib)
    for name, (backward, setup) in _FIT_AUTOGRAD.items():
        op = getattr(getattr(torch.ops, namespace), _FIT_BACKWARD_OP[name])
        torch.library.register_autograd(f"{namespace}::{name}", functools.partial(backward, op), setup_context=setup,
                                        lib=lib)
        if name == "dropout_add":
            torch.library.register_autograd(f"{namespace}::dropout_backward", functools.partial(_bw_dropout_backward, op),
                                            setup_context=_save_dropout_backward, lib=lib)
        else:
            torch.library.register_autograd(f"{namespace}::{_FIT_BACKWARD_OP[name]}", _no_second(name), lib=lib)
    _libs[key] = lib
    return names
