"""Embedding lookup and gradient, expert sort / dispatch / combine and its gradient, and
gradient clipping against plain implementations in 64 bits.

Tolerances follow from the operations, before any run: an output of type T is rounded once
(unit roundoff u_T, half the smallest subnormal near zero); a sum of m terms in fp32 is off by
at most (m + 2) * 2^-24 times the sum of the terms' magnitudes, products included.  Moves and
whole numbers are exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}
TYPES = [F32, F16, BF16]


def close(got, exact, terms=0, magnitude=None):
    """got (any type) against exact (fp64); magnitude: sum of the terms' absolute values."""
    bound = UNIT[got.dtype] * exact.abs() + TINY[got.dtype]
    if magnitude is not None:
        bound = bound + (terms + 2) * 2.0 ** -24 * magnitude * (1 + UNIT[got.dtype])
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, shape, dtype, pad=0, shift=0):
    """Normal values as a view with `pad` more columns a row, `shift` elements into its buffer."""
    rows, cols = shape
    buf = torch.full((rows * (cols + pad) + shift,), float("nan"), device="cuda", dtype=dtype)
    view = buf[shift:].view(rows, cols + pad)[:, :cols]
    view.copy_(torch.randn(shape, generator=g, device="cuda"))
    return view


def canvas(shape, dtype, pad=0, shift=0):
    """A view to write into and its whole buffer, filled with a canary."""
    rows, cols = shape
    buf = torch.full((rows * (cols + pad) + shift,), 7.0, device="cuda", dtype=dtype)
    return buf[shift:].view(rows, cols + pad)[:, :cols], buf


def untouched(view, buf):
    """Only the view's elements of its buffer were written."""
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
    return bool((buf[mask] == 7.0).all())


# ---- embedding ------------------------------------------------------------------------------

EMBED = [  # tokens, vocab, width, pad, shift
    (1, 1, 1, 0, 0), (1, 5, 64, 0, 0), (3, 7, 100, 0, 0), (33, 100, 8, 8, 0), (65, 50, 1031, 1, 1),
    (500, 1000, 256, 64, 8), (64, 300, 4100, 4, 2), (2049, 5, 24, 0, 4), (300, 70000, 36, 0, 0),
    (31, 9, 2, 2, 0), (4099, 31, 520, 0, 0), (700, 40, 333, 0, 0), (90, 60, 2050, 5, 3),
]


def token_ids(g, n, vocab, first, dtype):
    ids = torch.randint(-2, vocab + 2, (n,), generator=g, device="cuda") + first
    return ids.to(dtype)


@pytest.mark.parametrize("case", EMBED, ids=str)
@pytest.mark.parametrize("table_type", TYPES, ids=str)
@pytest.mark.parametrize("out_type", TYPES, ids=str)
def test_lookup(torch_cuda, dcopy, case, table_type, out_type):
    n, vocab, width, pad, shift = case
    g = gen(n + width)
    first, scale = (0, 1.0) if n % 2 else (1000, 11.3125)
    ids = token_ids(g, n, vocab, first, torch.int64 if n % 3 else torch.int32)
    table = randn(g, (vocab, width), table_type, pad, shift)
    out, buf = canvas((n, width), out_type, pad, shift)
    dcopy.embedding_lookup(out, table, ids, scale=scale, first_id=first)
    at = ids.long() - first
    known = (at >= 0) & (at < vocab)
    exact = table.double()[torch.where(known, at, 0)] * scale * known[:, None]
    close(out, exact, 1, exact.abs())
    assert untouched(out, buf)


def grad_exact(dout, at, vocab, scale):
    known = torch.nonzero((at >= 0) & (at < vocab))[:, 0]
    exact = torch.zeros(vocab, dout.shape[1], dtype=torch.float64, device="cuda")
    size = torch.zeros_like(exact)
    exact.index_add_(0, at[known], dout.double()[known] * scale)
    size.index_add_(0, at[known], dout.double()[known].abs() * abs(scale))
    return exact, size


@pytest.mark.parametrize("case", EMBED, ids=str)
@pytest.mark.parametrize("dout_type", TYPES, ids=str)
@pytest.mark.parametrize("grad_type", TYPES, ids=str)
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad(torch_cuda, dcopy, case, dout_type, grad_type, accumulate):
    n, vocab, width, pad, shift = case
    g = gen(3 * n + width)
    first, scale = (0, 1.0) if n % 2 else (-50, 0.328125)
    ids = token_ids(g, n, vocab, first, torch.int32 if n % 3 else torch.int64)
    dout = randn(g, (n, width), dout_type, pad, shift)
    grad, buf = canvas((vocab, width), grad_type, pad, shift)
    old = grad.clone()
    dcopy.embedding_grad(grad, dout, ids, scale=scale, first_id=first, accumulate=accumulate)
    exact, size = grad_exact(dout, ids.long() - first, vocab, scale)
    if accumulate:
        exact, size = exact + old.double(), size + old.double().abs()
    close(grad, exact, n, size)
    assert untouched(grad, buf)
    again, _ = canvas((vocab, width), grad_type, pad, shift)
    dcopy.embedding_grad(again, dout, ids, scale=scale, first_id=first, accumulate=accumulate)
    assert torch.equal(again, grad)  # the same bits


@pytest.mark.parametrize("ids", ["one", "two runs", "none", "every", "every back", "ends"])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 100, 511, 512, 513, 1024, 1025, 4096, 4097, 5000])
def test_embedding_grad_runs(torch_cuda, dcopy, ids, n):
    """Runs of equal ids that begin, cross and end at every place of the sorted list."""
    vocab, width = n + 3, 40
    k = torch.arange(n, device="cuda")
    ids = {"one": k * 0 + 2, "two runs": (k >= n // 3).long(), "none": k * 0 - 100, "every": k,
           "every back": n - 1 - k, "ends": torch.where(k % 2 == 0, 0, vocab - 1)}[ids]
    dout = randn(gen(n), (n, width), F32)
    grad = torch.full((vocab, width), float("nan"), device="cuda")
    dcopy.embedding_grad(grad, dout, ids)
    exact, size = grad_exact(dout, ids, vocab, 1.0)
    close(grad, exact, n, size)


@pytest.mark.parametrize("vocab", [1023, 1024, 1 << 20, (1 << 20) + 1, 3 << 20])
def test_embedding_grad_vocabularies(torch_cuda, dcopy, vocab):
    """Vocabularies around the digits of the sort: one, two and three passes."""
    g, n, width = gen(vocab), 9001, 8
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    ids[:4] = torch.tensor([0, vocab - 1, vocab, -1], device="cuda")
    dout = randn(g, (n, width), F32)
    grad = torch.empty((vocab, width), device="cuda")
    dcopy.embedding_grad(grad, dout, ids)
    exact, size = grad_exact(dout, ids, vocab, 1.0)
    close(grad, exact, n, size)


def test_embedding_nothing(torch_cuda, dcopy):
    """No tokens, no columns, no rows."""
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    table = torch.randn(5, 16, device="cuda")
    dcopy.embedding_lookup(torch.empty(0, 16, device="cuda"), table, ids)
    grad = torch.full((5, 16), 3.0, device="cuda")
    dcopy.embedding_grad(grad, torch.empty(0, 16, device="cuda"), ids, accumulate=True)
    assert bool((grad == 3.0).all())
    dcopy.embedding_grad(grad, torch.empty(0, 16, device="cuda"), ids)
    assert bool((grad == 0.0).all())
    out = torch.full((3, 16), 5.0, device="cuda")
    dcopy.embedding_lookup(out, torch.empty(0, 16, device="cuda"), ids.new_zeros(3))
    assert bool((out == 0.0).all())
    dcopy.embedding_lookup(torch.empty(3, 0, device="cuda"), torch.empty(4, 0, device="cuda"),
                           ids.new_zeros(3))


def test_embedding_ids_of_any_layout(torch_cuda, dcopy):
    """[batch, length] ids, a slice with a row pitch, and a strided vector."""
    table = torch.randn(50, 16, device="cuda")
    whole = torch.randint(0, 50, (6, 11), device="cuda")
    for ids in (whole, whole[:, 2:9], whole[1:5, 3]):
        out = torch.empty(ids.numel(), 16, device="cuda")
        dcopy.embedding_lookup(out, table, ids)
        assert torch.equal(out, table[ids.reshape(-1)])
        grad = torch.empty(50, 16, device="cuda")
        dcopy.embedding_grad(grad, out, ids)
        exact, size = grad_exact(out, ids.reshape(-1), 50, 1.0)
        close(grad, exact, ids.numel(), size)


def test_infinities_and_nan_stay_in_their_rows(torch_cuda, dcopy):
    table = torch.randn(8, 24, device="cuda", dtype=BF16)
    table[3], table[4, 5] = float("inf"), float("nan")
    ids = torch.tensor([0, 3, 4, -1, 2, 99], device="cuda")
    out = torch.empty(6, 24, device="cuda", dtype=BF16)
    dcopy.embedding_lookup(out, table, ids, scale=0.0)
    assert bool(out[1].isnan().all()) and bool(out[2, 5].isnan())
    assert bool((out[[0, 3, 4, 5]] == 0.0).all())
    grad = torch.empty(8, 24, device="cuda", dtype=BF16)
    dout = torch.ones(6, 24, device="cuda", dtype=BF16)
    dout[1], dout[3], dout[5] = float("inf"), float("nan"), float("nan")  # the last two: no row
    dcopy.embedding_grad(grad, dout, ids)
    assert bool(grad[3].isinf().all()) and bool(grad[[0, 1, 2, 4, 5, 6, 7]].isfinite().all())


def test_offsets_beyond_32_bits(torch_cuda, dcopy):
    """A table, a gradient and an expert buffer of more than 2^31 elements."""
    rows, width = 140000, 16384
    big = torch.empty((rows, width), dtype=BF16, device="cuda")
    far = torch.tensor([rows - 1, 5, rows - 2], device="cuda")
    big[far] = torch.randn(3, width, device="cuda").to(BF16)
    out = torch.empty(3, width, dtype=BF16, device="cuda")
    dcopy.embedding_lookup(out, big, far)
    assert torch.equal(out, big[far])
    dest = far.int().view(3, 1)
    dcopy.expert_combine(out.zero_(), big, dest)
    assert torch.equal(out, big[far])
    x = torch.randn(3, width, device="cuda").to(BF16)
    dcopy.expert_dispatch(big, x, dest)
    assert torch.equal(big[far], x)
    dw = torch.empty(3, 1, device="cuda")
    dy = torch.empty_like(big)
    dcopy.expert_combine_grad(dy, dw, x, big, dest, torch.full((3, 1), 2.0, device="cuda"))
    assert torch.equal(dy[far], x * 2)
    del dy
    dcopy.embedding_grad(big, x, far)
    assert torch.equal(big[far], x)
    assert int(torch.count_nonzero(big[6:rows - 2])) == 0
    norm = torch.empty(1, device="cuda")
    dcopy.clip_grad_norm(dcopy.GradList([big]), 1.0, norm)
    exact = float((x.double() ** 2).sum().sqrt())
    assert abs(norm.item() - exact) <= 40 * 2.0 ** -24 * exact


# ---- experts --------------------------------------------------------------------------------

ROUTES = [  # tokens, slots, experts, align, dropped
    (1, 1, 1, 1, 0.0), (1, 8, 8, 1, 0.0), (2, 3, 5, 4, 0.5), (64, 2, 64, 16, 0.0), (33, 4, 16, 7, 0.2),
    (1000, 6, 160, 1, 0.0), (3001, 2, 1023, 128, 0.1), (4096, 1, 2, 1, 0.0), (4097, 1, 3, 1, 1.0),
    (2500, 8, 60, 128, 0.3), (20000, 9, 33, 1, 0.01),
]


def routing(g, case, dtype=torch.int64):
    n, k, experts, align, drop = case
    ids = torch.randint(0, experts, (n, k), generator=g, device="cuda")
    ids[torch.rand(ids.shape, generator=g, device="cuda") < drop] = -1
    return ids.to(dtype)


def sort_exact(ids, experts, align, rows):
    flat = ids.reshape(-1).cpu().numpy().astype(np.int64)
    dest, source = np.full(flat.size, -1, np.int32), np.full(rows, -1, np.int32)
    offsets, at = [0], 0
    for e in range(experts):
        mine = np.flatnonzero(flat == e)
        dest[mine] = np.arange(at, at + mine.size)
        source[at:at + mine.size] = mine
        at += -(-mine.size // align) * align
        offsets.append(at)
    return dest.reshape(ids.shape), source, np.array(offsets, np.int32)


def sorted_route(dcopy, ids, case, extra=0):
    n, k, experts, align, _ = case
    rows = dcopy.expert_rows(n * k, experts, align) + extra
    dest = torch.full((n, k), 77, dtype=torch.int32, device="cuda")
    source = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    offsets = torch.full((experts + 1,), 77, dtype=torch.int32, device="cuda")
    dcopy.expert_sort(dest, source, offsets, ids, align=align)
    return dest, source, offsets


@pytest.mark.parametrize("case", ROUTES, ids=str)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
def test_expert_sort(torch_cuda, dcopy, case, dtype):
    ids = routing(gen(case[0]), case, dtype)
    dest, source, offsets = sorted_route(dcopy, ids, case, extra=5)
    d, s, o = sort_exact(ids, case[2], case[3], source.numel())
    assert np.array_equal(dest.cpu().numpy(), d)
    assert np.array_equal(source.cpu().numpy(), s)
    assert np.array_equal(offsets.cpu().numpy(), o)


def test_expert_sort_of_few_and_odd_choices(torch_cuda, dcopy):
    """No tokens; all choices on one expert; ids of a slice; ids outside the range."""
    case = (0, 2, 4, 16, 0.0)
    dest, source, offsets = sorted_route(dcopy, torch.empty(0, 2, dtype=torch.int64, device="cuda"),
                                         case, extra=3)
    assert offsets.tolist() == [0] * 5 and source.tolist() == [-1] * 3
    for ids in (torch.full((5000, 2), 3, device="cuda"),
                torch.randint(-5, 9, (3000, 5), device="cuda")[:, 1:3]):
        case = (ids.shape[0], 2, 4, 16, 0.0)
        dest, source, offsets = sorted_route(dcopy, ids, case)
        d, s, o = sort_exact(ids, 4, 16, source.numel())
        assert np.array_equal(dest.cpu().numpy(), d) and np.array_equal(source.cpu().numpy(), s)
        assert np.array_equal(offsets.cpu().numpy(), o)


def test_sorts_of_millions(torch_cuda, dcopy):
    """Lists beyond the smaller tiles of the sort: 5 M choices and 4.3 M tokens."""
    g = gen(17)
    ids = torch.randint(-1, 38, (2500000, 2), generator=g, device="cuda")
    dest, source, offsets = sorted_route(dcopy, ids, (2500000, 2, 37, 3, 0.0))
    flat = ids.view(-1)
    key = torch.where((flat >= 0) & (flat < 37), flat, 37)
    order = torch.argsort(key, stable=True)
    count = torch.bincount(key, minlength=38)
    first, padded = torch.cumsum(count, 0) - count, (count[:37] + 2) // 3 * 3
    ends = torch.cat([padded.new_zeros(1), torch.cumsum(padded, 0)])
    assert torch.equal(offsets.long(), ends)
    row = torch.arange(flat.numel(), device="cuda") - first[key[order]] + ends[key[order]]
    row = torch.where(key[order] < 37, row, -1)
    assert torch.equal(dest.view(-1)[order].long(), row)
    want = torch.full_like(source, -1)
    want[row[row >= 0]] = order[row >= 0].int()
    assert torch.equal(source, want)
    tokens, vocab = 4300000, 3001
    ids = torch.randint(-1, vocab + 1, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    dout = randn(g, (tokens, 4), F32)
    grad = torch.empty(vocab, 4, device="cuda")
    dcopy.embedding_grad(grad, dout, ids)
    exact, size = grad_exact(dout, ids.long(), vocab, 1.0)
    close(grad, exact, int(torch.bincount(ids.clamp(0, vocab - 1)).max()), size)


WIDTHS = [(1, 0, 0), (8, 0, 0), (17, 3, 5), (100, 4, 0), (257, 1, 1), (1024, 0, 0), (1030, 0, 0),
          (2056, 8, 8)]


@pytest.mark.parametrize("case", ROUTES[:10], ids=str)
@pytest.mark.parametrize("width", WIDTHS, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_there_and_back(torch_cuda, dcopy, case, width, dtype):
    n, k, experts, align, _ = case
    width, pad, shift = width
    g = gen(n * k + width)
    dest, source, _ = sorted_route(dcopy, routing(g, case), case)
    rows, kept = source.numel(), dest >= 0
    entry = source.long().clamp(min=0)
    held = (source >= 0)[:, None]
    x = randn(g, (n, width), dtype, pad, shift)
    w = randn(g, (n, k), F32, pad % 3, shift)

    out, buf = canvas((rows, width), dtype, pad, shift)
    dcopy.expert_dispatch(out, x, dest, source)
    assert torch.equal(out, torch.where(held, x[entry // k], 0.0)) and untouched(out, buf)

    out, buf = canvas((rows, width), dtype, pad, shift)
    dcopy.expert_dispatch(out, x, dest, source, w)
    exact = torch.where(held, x.double()[entry // k] * w.reshape(-1)[entry].double()[:, None], 0.0)
    close(out, exact, 1, exact.abs())
    assert untouched(out, buf)

    out, buf = canvas((rows, width), dtype, pad, shift)
    dcopy.expert_dispatch(out, x, dest)  # without source the other rows stay
    assert torch.equal(out, torch.where(held, x[entry // k], 7.0))

    y = randn(g, (rows, width), dtype, pad, shift)
    y[source < 0] = float("nan")  # rows of no token reach no result
    w2 = torch.where(kept, w, float("nan"))  # nor do weights of dropped choices
    terms = torch.where(kept[:, :, None], y.double()[dest.long().clamp(min=0)], 0.0)
    for weights in (None, w2):
        out, buf = canvas((n, width), dtype, pad, shift)
        dcopy.expert_combine(out, y, dest, weights)
        t = terms if weights is None else terms * torch.where(kept, w, 0.0).double()[:, :, None]
        close(out, t.sum(1), 2 * k, t.abs().sum(1))
        assert untouched(out, buf)

    dout = randn(g, (n, width), dtype, pad, shift)
    dy, buf = canvas((rows, width), dtype, pad, shift)
    dw, wbuf = canvas((n, k), F32, pad % 3, shift)
    dcopy.expert_combine_grad(dy, dw, dout, y, dest, w2, source)
    exact = torch.where(held, dout.double()[entry // k] * w.reshape(-1)[entry].double()[:, None], 0.0)
    close(dy, exact, 1, exact.abs())
    assert untouched(dy, buf) and untouched(dw, wbuf)
    t = terms * dout.double()[:, None, :]
    close(dw, t.sum(2), 2 * width, t.abs().sum(2))
    again = torch.empty_like(dw)
    dcopy.expert_combine_grad(dy, again, dout, y, dest, w2, source)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.float8_e4m3fn], ids=str)
def test_dispatch_moves_bytes(torch_cuda, dcopy, dtype):
    case = (100, 2, 8, 4, 0.1)
    dest, source, _ = sorted_route(dcopy, routing(gen(1), case), case)
    for width in (33, 128):
        x = torch.randint(-128, 128, (100, width), dtype=torch.int8, device="cuda")
        out = torch.full((source.numel(), width), 9, dtype=torch.int8, device="cuda")
        dcopy.expert_dispatch(out.view(dtype), x.view(dtype), dest, source)
        entry = source.long().clamp(min=0)
        assert torch.equal(out, torch.where((source >= 0)[:, None], x[entry // 2], 0))


def test_dispatch_keeps_every_bit(torch_cuda, dcopy):
    """All 16-bit patterns, NaN payloads among them, come out as they went in."""
    x = torch.arange(-32768, 32768, dtype=torch.int32, device="cuda").to(torch.int16).view(64, 1024)
    dest = torch.randperm(64, device="cuda", dtype=torch.int32).view(64, 1)
    out = torch.empty(64, 1024, dtype=torch.bfloat16, device="cuda")
    dcopy.expert_dispatch(out, x.view(torch.bfloat16), dest)
    assert torch.equal(out.view(torch.int16)[dest[:, 0].long()], x)


def test_many_slots(torch_cuda, dcopy):
    """More slots than a thread holds at once, and none at all."""
    case = (50, 37, 40, 1, 0.1)
    g = gen(8)
    dest, source, _ = sorted_route(dcopy, routing(g, case), case)
    y, dout = randn(g, (source.numel(), 72), BF16), randn(g, (50, 72), BF16)
    w = randn(g, (50, 37), F32)
    kept = dest >= 0
    terms = torch.where(kept[:, :, None], y.double()[dest.long().clamp(min=0)], 0.0)
    out = torch.empty(50, 72, dtype=BF16, device="cuda")
    dcopy.expert_combine(out, y, dest, w)
    t = terms * w.double()[:, :, None]
    close(out, t.sum(1), 74, t.abs().sum(1))
    dy, dw = torch.empty_like(y), torch.empty_like(w)
    dcopy.expert_combine_grad(dy, dw, dout, y, dest, w, source)
    t = terms * dout.double()[:, None, :]
    close(dw, t.sum(2), 144, t.abs().sum(2))
    dcopy.expert_combine(out, y, dest[:, :0].contiguous())
    assert bool((out == 0).all())


# ---- clipping -------------------------------------------------------------------------------

NORM = 40 * 2.0 ** -24  # 33 roundings of a thread's sum and product, its root and the result
COEF = NORM + 4 * 2.0 ** -24  # the sum with eps, the quotient, the product


def check_clip(dcopy, grads, outs, max_norm, eps=1e-6):
    before = [g.double() for g in grads]
    norm = torch.full((1,), -1.0, device="cuda")
    dcopy.clip_grad_norm(dcopy.GradList(grads, outs), max_norm, norm, eps=eps)
    exact = float(sum((b ** 2).sum() for b in before).sqrt()) if before else 0.0
    assert abs(norm.item() - exact) <= NORM * exact + 2.0 ** -149
    c = min(1.0, max_norm / (exact + eps)) if exact + eps else 1.0
    for b, o in zip(before, grads if outs is None else outs):
        err, e = (o.double() - b * c).abs(), (b * c).abs()
        assert bool((err <= (UNIT[o.dtype] + 2 * COEF) * e + TINY[o.dtype]).all())
    return norm.item(), c


@pytest.mark.parametrize("src", TYPES, ids=str)
@pytest.mark.parametrize("dst", TYPES + [None], ids=str)
@pytest.mark.parametrize("ratio", [0.25, 3.0])
def test_clip(torch_cuda, dcopy, src, dst, ratio):
    """Tensors of one element to several blocks' worth at odd places of a buffer."""
    g = gen(5)
    sizes = [1, 7, 8, 9, 4096, 4097, 16384, 16385, 100003, 0, 3, 300000]
    flat = torch.randn(sum(sizes), generator=g, device="cuda").to(src)
    grads = list(flat.split(sizes))
    outs = None if dst is None else list(torch.empty(sum(sizes) + 5, device="cuda", dtype=dst)[5:].split(sizes))
    check_clip(dcopy, grads, outs, ratio * sum(sizes) ** 0.5)


def test_clip_mixed_types_and_many(torch_cuda, dcopy):
    g = gen(6)
    grads = [torch.randn(1 + 37 * i % 5000, generator=g, device="cuda").to(TYPES[i % 3]) for i in range(700)]
    check_clip(dcopy, grads, None, 10.0)


def test_clip_in_place_without_need_changes_nothing(torch_cuda, dcopy):
    grads = [torch.randn(1000, device="cuda"), torch.randn(77, device="cuda").to(BF16)]
    copies = [g.clone() for g in grads]
    norm, _ = check_clip(dcopy, grads, None, 1e9)
    assert all(torch.equal(g, c) for g, c in zip(grads, copies))


@pytest.mark.parametrize("value", [0.0, float("inf"), float("nan")])
def test_clip_of_special_norms(torch_cuda, dcopy, value):
    """A zero norm leaves zeros; an infinite one gives c = 0 (and NaN where inf met it); NaN goes on."""
    g = torch.ones(5000, device="cuda") if value else torch.zeros(5000, device="cuda")
    g[4321] = value
    norm = torch.empty(1, device="cuda")
    dcopy.clip_grad_norm(dcopy.GradList([g]), 1.0, norm)
    if value == 0.0:
        assert norm.item() == 0.0 and bool((g == 0).all())
    elif value != value:
        assert bool(norm.isnan().all()) and bool(g.isnan().all())
    else:
        assert norm.item() == value and bool(g[4321].isnan()) and int(torch.count_nonzero(g)) == 1


def test_clip_of_large_and_small_values(torch_cuda, dcopy):
    """Squares that leave the range of fp32 are summed in range: 1e30 and 1e-30."""
    for scale in (1e30, 1e-30):
        g = torch.full((40000,), scale, device="cuda")
        norm = torch.empty(1, device="cuda")
        out = torch.empty_like(g)
        dcopy.clip_grad_norm(dcopy.GradList([g], [out]), 1.0, norm)
        exact = float(g[0].double()) * 200.0
        assert abs(norm.item() - exact) <= NORM * exact


def test_sum_and_clip_apart(torch_cuda, dcopy):
    """The two halves that ranks run around an addition of their sums."""
    a, b = torch.randn(5000, device="cuda"), torch.randn(3000, device="cuda")
    lists = [dcopy.GradList([a]), dcopy.GradList([b])]
    total = torch.zeros(2, dtype=torch.float64, device="cuda")
    want = float((a.double() ** 2).sum() + (b.double() ** 2).sum())
    for k, l in enumerate(lists):
        dcopy.grad_sum_squares(total[k:], l)
    both = total.sum(0, keepdim=True)
    assert abs(both.item() - want) <= 2 * NORM * want
    ea, norm = a.double() / (want ** 0.5 + 1e-6), torch.empty(1, device="cuda")
    for l in lists:
        dcopy.grad_clip(l, both, 1.0, norm)
    assert bool(((a.double() - ea).abs() <= (2.0 ** -24 + 2 * COEF) * ea.abs()).all())


# ---- gradients against differences -----------------------------------------------------------


def test_gradients_against_differences(torch_cuda, dcopy):
    """All maps are linear in each argument, so a central difference with any step is the
    derivative up to the rounding of the fp32 outputs it is taken of."""
    g = gen(11)
    n, k, vocab, width = 12, 3, 9, 6
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    table, seed = randn(g, (vocab, width), F32), randn(g, (n, width), F32)

    def lookup(t):
        out = torch.empty(n, width, device="cuda")
        dcopy.embedding_lookup(out, t, ids, scale=1.5)
        return (out.double() * seed.double()).sum()

    grad = torch.empty_like(table)
    dcopy.embedding_grad(grad, seed, ids, scale=1.5)
    case = (n, k, 4, 2, 0.2)
    dest, source, _ = sorted_route(dcopy, routing(g, case), case)
    y, w = randn(g, (source.numel(), width), F32), randn(g, (n, k), F32)

    def combine(y_, w_):
        out = torch.empty(n, width, device="cuda")
        dcopy.expert_combine(out, y_, dest, w_)
        return (out.double() * seed.double()).sum()

    dy, dw = torch.empty_like(y), torch.empty_like(w)
    dcopy.expert_combine_grad(dy, dw, seed, y, dest, w, source)
    for value, at, f in ((grad, table, lookup), (dy, y, lambda t: combine(t, w)),
                         (dw, w, lambda t: combine(y, t))):
        for i in range(at.numel()):
            step = torch.zeros_like(at).view(-1)
            step[i] = 1.0
            step = step.view_as(at)
            diff = float(f(at + step) - f(at - step)) / 2.0
            # n * width outputs of magnitude below 64, each within (k + 3) roundings.
            assert abs(value.reshape(-1)[i].item() - diff) <= n * width * 64 * (k + 3) * 2.0 ** -24


# ---- streams, graphs --------------------------------------------------------------------------


def test_side_stream_and_graph(torch_cuda, dcopy):
    """The calls on a stream of their own, workspaces from the allocator, and in a graph."""
    g = gen(3)
    n, k, vocab, width = 5000, 2, 600, 264
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    route = torch.randint(0, 16, (n, k), generator=g, device="cuda")
    x, w = randn(g, (n, width), F32), randn(g, (n, k), F32)
    rows = dcopy.expert_rows(n * k, 16)
    grad, out, norm = torch.empty(vocab, width, device="cuda"), torch.empty(n, width, device="cuda"), torch.empty(1, device="cuda")
    dest, source = torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    offsets, y = torch.empty(17, dtype=torch.int32, device="cuda"), torch.empty(rows, width, device="cuda")
    glist = dcopy.GradList([grad])

    def step(stream=None):
        dcopy.embedding_grad(grad, x, ids, stream=stream)
        dcopy.expert_sort(dest, source, offsets, route, stream=stream)
        dcopy.expert_dispatch(y, x, dest, source, stream=stream)
        dcopy.expert_combine(out, y, dest, w, stream=stream)
        dcopy.clip_grad_norm(glist, 1.0, norm, stream=stream)

    step()
    want = [t.clone() for t in (grad, out, norm, y)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t in (grad, out, norm, y):
        t.record_stream(side)
    step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (grad, out, norm, y)))
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (grad, out, norm, y)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in (grad, out, norm, y):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (grad, out, norm, y)))


def test_refusals_on_the_gpu(torch_cuda, dcopy):
    """Buffers that are too small, overlap or lie in host memory are refused before a launch."""
    table, ids = torch.randn(10, 32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")

    def refused(code, f, *a, **k):
        with pytest.raises(dcopy.DcopyError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value

    out = torch.empty(4, 32, device="cuda")
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.embedding_lookup, out[:3], table, ids)
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.embedding_lookup, out[:, :31], table, ids)
    refused(dcopy.ERR_DATATYPE_INVALID, dcopy.embedding_lookup, out.double(), table, ids)
    refused(dcopy.ERR_DATATYPE_INVALID, dcopy.embedding_lookup, out, table, ids.float())
    refused(dcopy.ERR_PARAM_INVALID, dcopy.embedding_lookup, table[2:6], table, ids)
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    refused(dcopy.ERR_PARAM_INVALID, dcopy.embedding_grad, table, out, ids, workspace=small)
    with pytest.raises(ValueError):
        dcopy.embedding_lookup(out, table, ids.cpu())
    with pytest.raises(ValueError):
        dcopy.embedding_lookup(out, table.t().contiguous().t(), ids)  # columns that are not dense
    i32 = dict(dtype=torch.int32, device="cuda")
    dest, source, offsets = torch.empty(4, 2, **i32), torch.empty(8, **i32), torch.empty(5, **i32)
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.expert_sort, dest, source[:7], offsets, dest.clone())
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.expert_sort, dest[:3], source, offsets, dest.clone())
    refused(dcopy.ERR_PARAM_INVALID, dcopy.expert_sort, dest, source, offsets, dest.clone(), align=0)
    refused(dcopy.ERR_UNSUPPORTED, dcopy.expert_sort, dest, source, torch.empty(2000, **i32), dest.clone())
    y = torch.empty(8, 32, device="cuda")
    refused(dcopy.ERR_DATATYPE_INVALID, dcopy.expert_combine, out, y.half(), dest)
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.expert_combine, out, y, dest, torch.ones(4, 3, device="cuda"))
    refused(dcopy.ERR_DATATYPE_INVALID, dcopy.expert_combine, out, y, dest, torch.ones(4, 2, device="cuda").half())
    refused(dcopy.ERR_SHAPE_INVALID, dcopy.expert_dispatch, y, out, dest, source[:5])
    refused(dcopy.ERR_PARAM_INVALID, dcopy.expert_dispatch, y, y[:4], dest)
    refused(dcopy.ERR_DATATYPE_INVALID, dcopy.GradList, [torch.ones(4, device="cuda", dtype=torch.float64)])
    base = torch.ones(100, device="cuda")
    refused(dcopy.ERR_PARAM_INVALID, dcopy.GradList, [base[:50]], [base[10:60]])
    refused(dcopy.ERR_PARAM_INVALID, dcopy.clip_grad_norm, dcopy.GradList([base]), float("nan"))


@pytest.mark.parametrize("n", [100, 5000])
def test_sort_in_place(torch_cuda, dcopy, n):
    """The routing written over the choices that it is made of."""
    case = (n, 3, 17, 4, 0.1)
    ids = routing(gen(n), case, torch.int32)
    d, s, o = sort_exact(ids, 17, 4, dcopy.expert_rows(3 * n, 17, 4))
    source = torch.empty(len(s), dtype=torch.int32, device="cuda")
    offsets = torch.empty(18, dtype=torch.int32, device="cuda")
    dcopy.expert_sort(ids, source, offsets, ids, align=4)
    assert np.array_equal(ids.cpu().numpy(), d) and np.array_equal(source.cpu().numpy(), s)
    assert np.array_equal(offsets.cpu().numpy(), o)


@pytest.mark.parametrize("n,width", [(2000, 24), (2000, 4096), (40, 4096)])
def test_weight_gradients_in_place_and_beside(torch_cuda, dcopy, n, width):
    """The weights' gradients written over the weights, and into columns beside them."""
    case = (n, 4, 16, 1, 0.1)
    g = gen(width)
    dest, source, _ = sorted_route(dcopy, routing(g, case), case)
    dout, y = randn(g, (n, width), BF16), randn(g, (source.numel(), width), BF16)
    both = randn(g, (n, 8), F32)
    w = both[:, :4].clone()
    dy, dw = torch.empty_like(y), torch.empty_like(w)
    dcopy.expert_combine_grad(dy, dw, dout, y, dest, w, source)
    got = torch.empty_like(dy)
    dcopy.expert_combine_grad(got, both[:, 4:], dout, y, dest, both[:, :4], source)
    assert torch.equal(got, dy) and torch.equal(both[:, 4:], dw) and torch.equal(both[:, :4], w)
    dcopy.expert_combine_grad(got, w, dout, y, dest, w, source)
    assert torch.equal(got, dy) and torch.equal(w, dw)


@pytest.mark.parametrize("shape", [(4, 0), (0, 4), (0,), (2, 3, 0)])
def test_empty_batches_of_any_shape(torch_cuda, dcopy, shape):
    """Batches without a token, with the zero in any place, as a training loop's last may be."""
    ids = torch.zeros(shape, dtype=torch.int64, device="cuda")
    table, x = torch.randn(9, 16, device="cuda"), torch.empty(*shape, 16, device="cuda")
    dcopy.embedding_lookup(x, table, ids, scale=2.0)
    grad = torch.full_like(table, 3.0)
    dcopy.embedding_grad(grad, x, ids)
    assert bool((grad == 0).all())
    chosen, w = ids[..., None].expand(*shape, 2).contiguous(), torch.empty(*shape, 2, device="cuda")
    dest = torch.empty(*shape, 2, dtype=torch.int32, device="cuda")
    source = torch.full((5,), 7, dtype=torch.int32, device="cuda")
    offsets = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    dcopy.expert_sort(dest, source, offsets, chosen, align=4)
    assert offsets.tolist() == [0] * 4 and source.tolist() == [-1] * 5
    rows, dw = torch.full((5, 16), 3.0, device="cuda"), torch.empty_like(w)
    dcopy.expert_dispatch(rows, x, dest, source)
    assert bool((rows == 0).all())
    dcopy.expert_combine(x, rows, dest, w)
    dy = torch.full_like(rows, 3.0)
    dcopy.expert_combine_grad(dy, dw, x, rows, dest, w, source)
    assert bool((dy == 0).all())


@pytest.mark.parametrize("n", [0, 1, 50])
def test_flat_routing_of_one_slot(torch_cuda, dcopy, n):
    """A router that picks one expert a token, its choices a vector; no tokens too."""
    g = gen(n)
    ids = torch.randint(0, 3, (n,), generator=g, device="cuda")
    dest, offsets = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    source = torch.empty(dcopy.expert_rows(n, 3, 4), dtype=torch.int32, device="cuda")
    dcopy.expert_sort(dest, source, offsets, ids, align=4)
    x, w = randn(g, (n, 8), F32), randn(g, (n, 1), F32)
    rows, out, dw = torch.empty(source.numel(), 8, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    dcopy.expert_dispatch(rows, x, dest, source, w)
    assert torch.equal(rows[dest.long()], x * w)
    dcopy.expert_dispatch(rows, x, dest, source)
    dcopy.expert_combine(out, rows, dest, w)
    assert torch.equal(out, x * w)
    dy = torch.empty_like(rows)
    dcopy.expert_combine_grad(dy, dw, x, rows, dest, w, source)
    assert torch.equal(dy[dest.long()], x * w)
    exact = (x.double() ** 2).sum(1, keepdim=True)
    close(dw, exact, 16, exact)


@pytest.mark.parametrize("n", [100, 600, 5000])
def test_ids_at_the_ends_of_the_range(torch_cuda, dcopy, n):
    """Ids and first ids as far apart as 64 bits allow belong nowhere but where they do."""
    top = (1 << 63) - 1
    odd = torch.tensor([top, -top - 1, top - 1, -top, 0, -1, top - 3, -top + 2], device="cuda")
    ids = odd[torch.arange(n, device="cuda") % 8]
    table, dout = torch.randn(4, 8, device="cuda"), torch.randn(n, 8, device="cuda")
    for first, rows in ((top - 3, {0: 3, 2: 2, 6: 0}), (-top - 1, {1: 0, 3: 1, 7: 3}), (-1, {4: 1, 5: 0})):
        at = torch.full((8,), -1, device="cuda")
        for k, row in rows.items():
            at[k] = row
        at = at[torch.arange(n, device="cuda") % 8]
        out = torch.empty(n, 8, device="cuda")
        dcopy.embedding_lookup(out, table, ids, first_id=first)
        assert torch.equal(out, torch.where((at >= 0)[:, None], table[at.clamp(min=0)], 0.0))
        grad = torch.empty_like(table)
        dcopy.embedding_grad(grad, dout, ids, first_id=first)
        exact, size = grad_exact(dout, at, 4, 1.0)
        close(grad, exact, n, size)


@pytest.mark.parametrize("n", [700, 1500, 4096, 4097, 9001])
@pytest.mark.parametrize("vocab", [510, 511, 512, (1 << 18) - 1, 1 << 18, (1 << 18) + 1, (1 << 27) - 1, 1 << 27])
def test_embedding_grad_where_passes_begin(torch_cuda, dcopy, vocab, n):
    """Vocabularies on both sides of one, two, three and four passes of the sort (the key that
    belongs nowhere is `vocab` itself, so 511 fills nine bits), of one tile and of several."""
    g = gen(vocab + n)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    ids[::3] = torch.randint(max(0, vocab - 600), vocab + 1, (len(ids[::3]),), generator=g, device="cuda")
    ids[:4] = torch.tensor([0, vocab - 1, vocab, -1], device="cuda")
    if vocab > 1 << 20:  # wide tables: what they held stays, and only rows of tokens are looked at
        dout, grad = randn(g, (n, 2), BF16), torch.full((vocab, 2), 2.0, device="cuda", dtype=BF16)
        dcopy.embedding_grad(grad, dout, ids, accumulate=True)
        known = (ids >= 0) & (ids < vocab)
        rows, at = torch.unique(ids[known], return_inverse=True)
        exact, size = grad_exact(dout[known], at, rows.numel(), 1.0)
        close(grad[rows], exact + 2.0, n, size + 2.0)
        assert int((grad != 2.0).any(1).sum()) <= rows.numel()
        return
    dout, grad = randn(g, (n, 8), F32), torch.empty((vocab, 8), device="cuda")
    dcopy.embedding_grad(grad, dout, ids)
    exact, size = grad_exact(dout, ids, vocab, 1.0)
    close(grad, exact, n, size)


def test_a_routing_is_needed(torch_cuda, dcopy):
    """No dest is an error, not a routing without slots."""
    x, rows = torch.ones(4, 8, device="cuda"), torch.ones(6, 8, device="cuda")
    source, w = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    with pytest.raises(ValueError):
        dcopy.expert_dispatch(rows, x, None, source)
    with pytest.raises(ValueError):
        dcopy.expert_combine(x, rows, None)
    with pytest.raises(ValueError):
        dcopy.expert_combine_grad(torch.empty_like(rows), w.clone(), x, rows, None, w, source)
    assert bool((x == 1).all()) and bool((rows == 1).all())


def test_accumulate_is_a_truth_value(torch_cuda, dcopy):
    """What has none raises its own error before anything is written."""
    grad, dout = torch.ones(4, 8, device="cuda"), torch.ones(3, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="ambiguous"):
        dcopy.embedding_grad(grad, dout, ids, accumulate=np.ones(2))
    assert bool((grad == 1).all())
    dcopy.embedding_grad(grad, dout, ids, accumulate=np.bool_(True))
    assert bool((grad[0] == 4).all()) and bool((grad[1:] == 1).all())
