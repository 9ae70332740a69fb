"""The differentiable torch.ops.dcopy operators of language models: shapes without a GPU,
gradients against autograd through torch's own indexing, and the training example."""
import sys

import pytest
import torch

from conftest import ROOT


@pytest.fixture(scope="module")
def ops(dcopy):
    from dcopy import torch_ops  # noqa: F401  (registers torch.ops.dcopy.*)
    return torch.ops.dcopy


def test_fake_shapes_without_a_gpu(ops):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        table, ids = torch.empty(50, 24), torch.empty(3, 7, dtype=torch.int64)
        assert list(ops.embedding(table, ids).shape) == [3, 7, 24]
        assert list(ops.embedding_backward(torch.empty(3, 7, 24), ids, 50).shape) == [50, 24]
        dest, source, offsets = ops.expert_sort(torch.empty(10, 2, dtype=torch.int64), 4, 16)
        assert [list(t.shape) for t in (dest, source, offsets)] == [[10, 2], [80], [5]]
        rows = ops.expert_dispatch(torch.empty(10, 24), dest, source)
        assert list(rows.shape) == [80, 24]
        assert list(ops.expert_combine(rows, dest, source, torch.empty(10, 2)).shape) == [10, 24]


def _route(ops):
    ids = torch.randint(-1, 4, (30, 3), device="cuda")
    return ids, *ops.expert_sort(ids, 4, 8)


@pytest.mark.gpu
def test_gradients_match_autograd(ops, torch_cuda):
    """fp32 on sums of at most 30 terms of magnitude below 100: 32 * 100 * 2^-24."""
    tol = dict(rtol=0, atol=32 * 100 * 2.0 ** -24)
    torch.manual_seed(0)
    ids = torch.randint(0, 9, (5, 6), device="cuda")
    for expand in (False, True):
        table = torch.randn(9, 20, device="cuda", requires_grad=True)
        seed = torch.randn(5, 6, 1, device="cuda").expand(5, 6, 20)  # a gradient of stride 0
        seed = seed if expand else torch.randn(5, 6, 20, device="cuda")
        got, = torch.autograd.grad(ops.embedding(table, ids, 1.5), table, seed)
        want, = torch.autograd.grad(table[ids] * 1.5, table, seed)
        torch.testing.assert_close(got, want, **tol)
    chosen, dest, source, offsets = _route(ops)
    kept = (dest >= 0)[:, :, None]
    x = torch.randn(30, 20, device="cuda", requires_grad=True)
    w = torch.randn(30, 3, device="cuda", requires_grad=True)
    seed = torch.randn(30, 20, device="cuda")

    def plain(x, w):
        rows = torch.where((source >= 0)[:, None], x[source.long().clamp(min=0) // 3], 0.0)
        back = torch.where(kept, (rows * 1.25)[dest.long().clamp(min=0)], 0.0)
        return (back if w is None else back * w[:, :, None]).sum(1)

    def ours(x, w):
        return ops.expert_combine(ops.expert_dispatch(x, dest, source) * 1.25, dest, source, w)

    for weights in (w, None):
        args = (x, w) if weights is not None else (x,)
        got = torch.autograd.grad(ours(x, weights), args, seed)
        want = torch.autograd.grad(plain(x, weights), args, seed)
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, **tol)


@pytest.mark.gpu
def test_weights_of_the_rows_type(ops, torch_cuda):
    """A router in bf16: its weights count as the fp32 values they stand for, and their
    gradient comes back in bf16."""
    chosen, dest, source, _ = _route(ops)
    y = torch.randn(source.numel(), 20, device="cuda").bfloat16()
    w = torch.randn(30, 3, device="cuda").bfloat16().requires_grad_()
    seed = torch.randn(30, 20, device="cuda").bfloat16()
    out = ops.expert_combine(y, dest, source, w)
    assert torch.equal(out, ops.expert_combine(y, dest, source, w.detach().float()))
    got, = torch.autograd.grad(out, w, seed)
    _, want = ops.expert_combine_backward(seed, y, dest, source, w.detach().float())
    assert got.dtype == torch.bfloat16 and torch.equal(got, want.bfloat16())


@pytest.mark.gpu
def test_opcheck(ops, torch_cuda):
    chosen, dest, source, _ = _route(ops)
    x, w = torch.randn(30, 20, device="cuda"), torch.randn(30, 3, device="cuda")
    y = ops.expert_dispatch(x, dest, source)
    which = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(ops.embedding, (torch.randn(9, 8, device="cuda"), chosen.clamp(min=0)),
                          test_utils=which)
    torch.library.opcheck(ops.expert_sort, (chosen, 4, 8), test_utils=which[:2])
    torch.library.opcheck(ops.expert_dispatch, (x, dest, source), test_utils=which)
    torch.library.opcheck(ops.expert_combine, (y, dest, source, w), test_utils=which)


@pytest.mark.gpu
def test_training_example(torch_cuda):
    """The example's losses follow the plain model's: the first step within fp32 rounding
    (products of width 256 in the library's and torch's order: 1e-4), later ones within 1e-2,
    and training lowers the loss."""
    sys.path.insert(0, str(ROOT / "examples"))
    import moe_step
    a, b = moe_step.train(8, plain=False), moe_step.train(8, plain=True)
    assert abs(a[0][0] - b[0][0]) <= 1e-4 * b[0][0] and abs(a[0][1] - b[0][1]) <= 1e-4 * b[0][1]
    assert all(abs(x[0] - y[0]) <= 1e-2 * y[0] for x, y in zip(a, b))
    assert a[-1][0] < a[0][0]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 3), (0,), (4, 0)])
@pytest.mark.parametrize("width", [0, 8])
def test_embedding_without_elements(ops, torch_cuda, shape, width):
    """Tables without columns and batches without tokens, there and back."""
    ids = torch.zeros(shape, dtype=torch.int64, device="cuda")
    table = torch.randn(5, width, device="cuda", requires_grad=True)
    out = ops.embedding(table, ids, 2.0)
    assert torch.equal(out, table[ids] * 2.0)
    grad, = torch.autograd.grad(out.sum(), table)
    want = torch.zeros(5, width, device="cuda")
    want[:1] = 2.0 * ids.numel()
    assert torch.equal(grad, want)
