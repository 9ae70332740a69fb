"""The model operators on streams other than torch's current one: whose memory their
workspaces take, and how long a gradient list's table is kept."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BUSY = 40_000_000  # clock cycles that a stream is kept busy, some 20 ms


def pool_bytes(stream):
    """Bytes of the allocator's segments that belong to a stream."""
    return sum(s["total_size"] for s in torch.cuda.memory_snapshot()
               if s["stream"] == stream.cuda_stream)


@pytest.fixture
def fresh_stream(torch_cuda):
    """A stream without memory of its own."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for _ in range(32):
        side = torch.cuda.Stream()
        if pool_bytes(side) == 0:
            return side
    pytest.fail("every stream holds memory")


def calls(dcopy, tokens=5000, vocab=600, width=264, experts=16):
    """Inputs and outputs of the two calls that take a workspace, and the calls."""
    g = torch.Generator(device="cuda").manual_seed(21)
    whole = dict(dtype=torch.int32, device="cuda")
    ids = torch.randint(-1, vocab, (tokens,), generator=g, device="cuda")
    chosen = torch.randint(-1, experts, (tokens, 2), generator=g, device="cuda")
    dout = torch.randn(tokens, width, generator=g, device="cuda")
    outs = [torch.empty(vocab, width, device="cuda"), torch.empty(tokens, 2, **whole),
            torch.empty(dcopy.expert_rows(2 * tokens, experts, 8), **whole),
            torch.empty(experts + 1, **whole)]

    def run(stream=None):
        dcopy.embedding_grad(outs[0], dout, ids, stream=stream)
        dcopy.expert_sort(*outs[1:], chosen, align=8, stream=stream)

    return outs, run


@pytest.mark.parametrize("as_number", [False, True])
def test_workspaces_are_the_given_streams(dcopy, fresh_stream, as_number):
    """A workspace that is not given comes from the pool of the stream the call runs on: what
    kernels pending on the current stream still do with memory freed there does not reach it."""
    side = fresh_stream
    outs, run = calls(dcopy)
    run()
    want = [t.clone() for t in outs]
    for t in outs:
        t.fill_(-7)
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda._sleep(BUSY)
    scratch = [torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(8)]
    del scratch  # free for the current stream, whose fills are still to come
    before = torch.cuda.current_stream().cuda_stream
    run(side.cuda_stream if as_number else side)
    assert torch.cuda.current_stream().cuda_stream == before
    assert pool_bytes(side) > 0
    side.synchronize()
    got = [t.clone() for t in outs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def span(t):
    return t.data_ptr(), t.data_ptr() + t.nbytes


@pytest.mark.parametrize("given", ["stream", "number", "current"])
@pytest.mark.parametrize("call", ["clip_grad_norm", "grad_sum_squares", "grad_clip"])
def test_a_dropped_list_is_kept_until_its_streams_are_done(torch_cuda, dcopy, given, call):
    """A list dropped while another stream's call on it is still pending: the memory of its
    table, and of outputs that only the list held, goes to nobody else before."""
    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(5)
    grads = [torch.randn(n, generator=g, device="cuda") for n in (100003, 7, 4096, 50000)]
    want = [t.clone() for t in grads]
    norm, total = torch.empty(1, device="cuda"), torch.empty(1, dtype=torch.float64, device="cuda")
    args = {"clip_grad_norm": (1.0, norm), "grad_clip": (total, 1.0, norm)}.get(call)

    def run(grads, outs, **stream):
        held = dcopy.GradList(grads, outs)
        if call == "grad_sum_squares":
            dcopy.grad_sum_squares(total, held, **stream)
        else:
            dcopy.__dict__[call](held, *args, **stream)
        return held

    total.fill_(9.0)
    run(want, None)
    torch.cuda.synchronize()
    expected = float(total if call == "grad_sum_squares" else norm)
    norm.zero_()
    if call == "grad_sum_squares":
        total.zero_()
    outs = [torch.empty_like(t) for t in grads]
    for t in grads:
        t.record_stream(side)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(5 * BUSY)
    if given == "current":
        held = dcopy.GradList(grads, outs)
        with torch.cuda.stream(side):
            if call == "grad_sum_squares":
                dcopy.grad_sum_squares(total, held)
            else:
                dcopy.__dict__[call](held, *args)
    else:
        held = run(grads, outs, stream=side if given == "stream" else side.cuda_stream)
    kept = [held._space] + outs
    taken, sizes = [span(t) for t in kept], [t.nbytes for t in kept]
    del kept, held, outs
    others = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(8)]
    assert not side.query()  # still busy
    assert all(b <= lo or hi <= a for a, b in taken for lo, hi in map(span, others))
    side.synchronize()
    assert float(total if call == "grad_sum_squares" else norm) == expected


def test_a_list_lives_on_the_stream_it_is_built_on(dcopy, fresh_stream):
    """The table's memory is of the given stream's pool, as the copy that fills it runs there."""
    grads = [torch.ones(1000, device="cuda")]
    held = dcopy.GradList(grads, stream=fresh_stream)
    assert pool_bytes(fresh_stream) >= held._space.nbytes
    norm = torch.empty(1, device="cuda")
    dcopy.clip_grad_norm(held, 1.0, norm)
    assert abs(norm.item() - 1000 ** 0.5) <= 40 * 2.0 ** -24 * 1000 ** 0.5


def test_given_streams_inside_a_graph(torch_cuda, dcopy):
    """A captured step that forks to a stream of its own: workspaces come from the graph's
    memory, and a list used there stays usable outside."""
    outs, run = calls(dcopy)
    grads = [torch.randn(5000, device="cuda"), torch.randn(77, device="cuda")]
    clipped, norm = [torch.empty_like(g) for g in grads], torch.empty(1, device="cuda")
    held = dcopy.GradList(grads, clipped)
    run()
    dcopy.clip_grad_norm(held, 1.0, norm)
    everything = outs + clipped + [norm]
    want = [t.clone() for t in everything]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        run(side)
        dcopy.clip_grad_norm(held, 1.0, norm, stream=side)
        torch.cuda.current_stream().wait_stream(side)
    for t in everything:
        t.fill_(-7)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, everything))
    norm.zero_()
    dcopy.clip_grad_norm(held, 1.0, norm)
    assert torch.equal(norm, want[-1])
