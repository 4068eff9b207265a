"""LayerCache8 calls with stream=: workspaces and results are memory of that stream, so nothing else is given them while the
call may still be running, and the results are those of the current stream."""
import pytest

pytestmark = pytest.mark.gpu

N = 2000


@pytest.fixture()
def held(la, cuda):
    import torch

    gen = torch.Generator(device=cuda).manual_seed(5)
    cache = la.LayerCache8(la.MODE_E4M3BLK, 2, 64, N + 64, device=cuda)
    k, v = (torch.randn(N, 2, 64, generator=gen, device=cuda).half() for _ in range(2))
    cache.append(k, v)
    q = torch.randn(8, 8, 64, generator=gen, device=cuda).half()
    chunk = torch.randn(200, 8, 64, generator=gen, device=cuda).half()
    lse = torch.empty(8, 8, device=cuda)
    cache.verify(q, N - 8, lse=lse)
    w = torch.rand(2, N, generator=gen, device=cuda)
    dst = la.LayerCache8(la.MODE_E4M3BLK, 2, 64, 512, device=cuda)
    torch.cuda.synchronize()
    return {
        "verify": lambda s: cache.verify(q, N - 8, splits=5, stream=s),
        "prefill": lambda s: cache.prefill(chunk, N - 200, stream=s),
        "read": lambda s: cache.read(100, 700, stream=s),
        "weights": lambda s: cache.key_weights(q, lse, N - 8, stream=s),
        "evict": lambda s: cache.evict(w, 400, 4, 32, dst, stream=s),
        "select": lambda s: la.evict_select(w, N, 400, 4, 32, stream=s),
    }, cache


CALLS = ["verify", "prefill", "read", "weights", "evict", "select"]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("as_handle", [False, True])
def test_results(la, cuda, held, name, as_handle):
    import torch

    call = held[0][name]
    side = torch.cuda.Stream()
    want = call(None)
    torch.cuda.synchronize()
    for s in (side, torch.cuda.default_stream()):
        got = call(s.cuda_stream if as_handle else s)
        assert torch.cuda.current_stream() == torch.cuda.default_stream()
        s.synchronize()
        la.sync(s)
        for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, want))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", CALLS)
def test_results_are_the_streams_memory(cuda, held, name):
    """Dropped results: the current stream is not given their memory, nor is the other stream while the current one, which
    may still read them, is busy."""
    import torch

    call = held[0][name]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)   # some 10 ms of the current stream
    got = call(side)
    got = got if isinstance(got, tuple) else (got,)
    like = [(x.shape, x.dtype, x.data_ptr()) for x in got]
    del got
    for shape, dtype, address in like:
        assert torch.empty(shape, dtype=dtype, device=cuda).data_ptr() != address
        with torch.cuda.stream(side):
            assert torch.empty(shape, dtype=dtype, device=cuda).data_ptr() != address
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", ["verify", "prefill"])
def test_workspace_is_the_streams_memory(la, cuda, held, monkeypatch, name):
    """The workspace that a call makes is free again when it returns, but for its own stream only."""
    import torch

    calls, cache = held
    seen = []

    def watch(owner, attribute, at):
        real = getattr(owner, attribute)
        monkeypatch.setattr(owner, attribute, lambda *a: seen.append((a[at], a[at + 1])) or real(*a))

    watch(cache, "_attention", 11)
    watch(la.lib(), "lfm3a_kv8_prefill", 9)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls[name](side)
    (address, size), = seen
    assert size > 0
    assert torch.empty(size, dtype=torch.uint8, device=cuda).data_ptr() != address
    torch.cuda.synchronize()
