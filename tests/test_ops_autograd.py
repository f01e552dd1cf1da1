"""vectordb_amd.ops and autograd: gradients are not lost in silence, and what is written in place is noticed."""

import pytest
import torch

from vectordb_amd import ops


def arguments(device):
    """The calls, with the names of their tensors that can require a gradient."""
    x, u, lists = torch.zeros(4, 8, device=device), torch.zeros(4, device=device), torch.zeros(4, 2, device=device)
    at, rows = torch.zeros(4, dtype=torch.int64, device=device), torch.zeros(4, 2, dtype=torch.int64, device=device)
    return [
        (ops.lookup, dict(table=x, rows=at, out=x.clone()), ("table", "out")),
        (ops.lookup_grad, dict(grad=x, rows=at, n_rows=5, out=torch.zeros(5, 8, device=device)), ("grad", "out")),
        (ops.distill, dict(scores=x, teacher=lists, rows=rows, teacher_lse=u), ("scores", "teacher", "teacher_lse")),
        (ops.distill_grad, dict(scores=x, teacher=lists, rows=rows, stats=lists.clone(), grad_loss=u, out=x.clone()),
         ("scores", "teacher", "stats", "grad_loss", "out")),
        (ops.distill_step, dict(scores=x, teacher=lists, rows=rows, grad_loss=u, out=x.clone()), ("scores", "teacher", "grad_loss", "out")),
        (ops.sample, dict(scores=x, uniforms=u, temperature=u.clone() + 1), ("scores", "temperature")),
    ]


def test_first_tensors_that_require_a_gradient_are_refused():
    """Before anything else is asked of them, so without a GPU too."""
    for call, args, names in arguments("cpu"):
        args = {**args, names[0]: args[names[0]].clone().requires_grad_()}
        others = {k: v for k, v in args.items() if k != "out"}
        if call in (ops.lookup, ops.lookup_grad):          # row numbers come first
            continue
        with pytest.raises(ValueError, match="requires a gradient"):
            call(**others)


@pytest.mark.gpu
def test_tensors_that_require_a_gradient_are_refused(native):
    for call, args, names in arguments("cuda"):
        call(**args)
        for name in names:
            asked = {**args, name: args[name].clone().requires_grad_()}
            with pytest.raises(ValueError, match=f"{name} requires a gradient"):
                call(**asked)
            with torch.no_grad():
                call(**asked)


@pytest.mark.gpu
def test_gradients_of_a_function(native):
    """The calls inside a torch.autograd.Function, where gradients are not recorded: the gradient reaches the table."""
    class Rows(torch.autograd.Function):
        @staticmethod
        def forward(ctx, table, at):
            ctx.save_for_backward(at)
            ctx.n_rows = table.shape[0]
            return ops.lookup(table, at, scale=0.5)

        @staticmethod
        def backward(ctx, grad):
            return ops.lookup_grad(grad, ctx.saved_tensors[0], ctx.n_rows, scale=0.5), None

    table = torch.randn(30, 8, device="cuda", requires_grad=True)
    at = torch.randint(0, 30, (50,), device="cuda")
    weight = torch.randint(-3, 4, (50, 8), device="cuda").float()
    (Rows.apply(table, at) * weight).sum().backward()
    want = torch.zeros(30, 8, device="cuda").index_add_(0, at, 0.5 * weight)
    assert torch.equal(table.grad, want)                   # multiples of 1/2: exact


@pytest.mark.gpu
def test_writing_to_out_is_noticed(native):
    """A tensor that autograd has kept, overwritten by a call, makes the backward pass fail as after any in-place operation."""
    for call, args, names in arguments("cuda"):
        if "out" not in args:
            continue
        factor = torch.ones_like(args["out"], requires_grad=True)
        kept = (factor * args["out"]).sum()
        call(**args)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    x = torch.zeros(4, 8, device="cuda")
    factor = torch.ones_like(x, requires_grad=True)
    kept = (factor * x).sum()
    call, args, _ = arguments("cuda")[4]
    call(**{**args, "scores": x, "out": x})                # in place of the scores
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
