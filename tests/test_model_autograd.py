"""What the differentiable torch.ops.dcopy operators keep between forward and backward, and
their shapes under tracing.  No GPU: fake tensors run the same autograd code."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(scope="module")
def ops(dcopy):
    from dcopy import torch_ops  # noqa: F401  (registers torch.ops.dcopy.*)
    return torch.ops.dcopy


def operators(ops, weighted):
    """Each operator's output, and the tensors of whole numbers that its gradient reads again."""
    ids = torch.zeros(7, dtype=torch.int64)
    dest, source = torch.zeros(10, 2, dtype=torch.int32), torch.zeros(80, dtype=torch.int32)
    weights = torch.empty(10, 2, requires_grad=True) if weighted else None
    table = torch.empty(50, 24, requires_grad=True)
    x, y = torch.empty(10, 24, requires_grad=True), torch.empty(80, 24, requires_grad=True)
    return {"embedding": (ops.embedding(table, ids), (ids,)),
            "expert_dispatch": (ops.expert_dispatch(x, dest, source), (dest, source)),
            "expert_combine": (ops.expert_combine(y, dest, source, weights), (dest, source))}


@pytest.mark.parametrize("name,weighted,which", [
    ("embedding", False, 0), ("expert_dispatch", False, 0), ("expert_dispatch", False, 1),
    ("expert_combine", False, 0), ("expert_combine", False, 1), ("expert_combine", True, 0),
    ("expert_combine", True, 1)])
def test_changed_indices_are_noticed(ops, name, weighted, which):
    """Ids or a routing overwritten before the backward pass raise, as they do in torch's own
    indexing, and give no gradient of the new contents."""
    with FakeTensorMode():
        out, kept = operators(ops, weighted)[name]
        kept[which].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


@pytest.mark.parametrize("weighted,count", [(False, 1 + 2 + 2), (True, 1 + 2 + 4)])
def test_hooks_see_what_is_kept(ops, weighted, count):
    """Saved-tensor hooks (offloading, recomputation) get every tensor kept for the backward:
    the ids; dest and source; dest and source, and y and the weights where there are weights."""
    with FakeTensorMode():
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
            outs = operators(ops, weighted)
        assert len(seen) == count
        for out, _ in outs.values():
            out.sum().backward()


@pytest.mark.parametrize("align", [1, 16])
def test_token_counts_stay_symbolic(dcopy, ops, align):
    """Traced with dynamic shapes, the rows of a routing follow the token count: nothing turns
    it into the number of the example."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(chosen, x):
        dest, source, offsets = ops.expert_sort(chosen, 4, align)
        return ops.expert_combine(ops.expert_dispatch(x, dest, source), dest, source), source

    traced = make_fx(step, tracing_mode="symbolic")(torch.zeros(10, 2, dtype=torch.int64),
                                                    torch.zeros(10, 8))
    rows = next(n for n in traced.graph.nodes if "expert_dispatch" in str(n.target)).meta["val"].shape[0]
    assert isinstance(rows, torch.SymInt)
    expr = rows.node.expr
    assert len(expr.free_symbols) == 2  # tokens and slots
    for tokens, slots in ((5, 3), (1, 1), (300, 2)):
        sizes = dict(zip(expr.free_symbols, (tokens, slots)))
        assert int(expr.subs(sizes)) == dcopy.expert_rows(tokens * slots, 4, align)


@pytest.mark.gpu
def test_opcheck_with_dynamic_shapes(ops, torch_cuda):
    """The operators traced for all sizes give what they give when called."""
    from torch.library import opcheck
    chosen = torch.randint(-1, 4, (30, 3), device="cuda")
    dest, source, _ = ops.expert_sort(chosen, 4, 8)
    x = torch.randn(30, 20, device="cuda", requires_grad=True)
    w = torch.randn(30, 3, device="cuda", requires_grad=True)
    y = torch.randn(source.numel(), 20, device="cuda", requires_grad=True)
    table = torch.randn(9, 8, device="cuda", requires_grad=True)
    for op, args in ((ops.embedding, (table, chosen)), (ops.expert_sort, (chosen, 4, 8)),
                     (ops.expert_dispatch, (x, dest, source)), (ops.expert_combine, (y, dest, source, w)),
                     (ops.expert_combine, (y, dest, source))):
        opcheck(op, args, test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                      "test_aot_dispatch_dynamic"))
