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
