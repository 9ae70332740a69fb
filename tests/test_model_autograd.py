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
