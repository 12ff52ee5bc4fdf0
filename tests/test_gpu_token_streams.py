"""Token operators on a stream that is not the current one: results and
workspaces come from that stream's memory.  (A block that the current stream
has freed may still be written by kernels queued there.)"""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def owner(t):
    """Handle of the stream whose memory holds the tensor."""
    at = t.data_ptr()
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= at < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not the allocator's")


def calls():
    """name -> (call of a stream that gives its results, whether it takes a workspace)"""
    x = torch.randn((2, 3000, 64), device="cuda").to(F16)
    blobs = x.transpose(1, 2).contiguous()
    tok = x.view(2, 3000, 2, 32)
    pos = torch.zeros((1, 3000, 2), dtype=torch.int32, device="cuda")
    norm, planes, rot = nhip.GroupNorm(8, 64), nhip.GroupNorm(8, 64, blobs=True), nhip.Rotary(32, (8, 8))
    q, k = torch.randn((2, 1, 8, 64), device="cuda").to(F16), torch.randn((2, 4000, 2, 64), device="cuda").to(F16)
    cache = nhip.KvCache8(128, 2, 64, 64)
    table = torch.arange(128, dtype=torch.int32, device="cuda").view(2, 64)
    zero, full = (torch.full((2,), n, dtype=torch.int32, device="cuda") for n in (0, 4000))
    cache.append(k, k, table, zero)
    return {
        "norm": (lambda s: norm.forward(x, stream=s), True),
        "norm blobs": (lambda s: planes.forward(blobs, stream=s), True),
        "rotary": (lambda s: rot.forward(tok, pos, stream=s), False),
        "cross": (lambda s: nhip.cross_attention(q, k, k, stream=s), True),
        "read": (lambda s: cache.read(table, zero, 300, F16, stream=s), False),
        "cached": (lambda s: cache.attention(q, table, full, stream=s), True),
    }


@pytest.mark.parametrize("name", ["norm", "norm blobs", "rotary", "cross", "read", "cached"])
def test_memory_of_the_stream(name, nhip_env, monkeypatch):
    nhip_env.setenv("NHIP_NORM_ONE", "0")  # two launches: a workspace
    call, scratch = calls()[name]
    want = call(None)
    places = []

    def spy(*args):
        r = take(*args)
        if r[0] is not None:
            places.append(owner(r[0]))
        return r

    take = nhip._scratch
    monkeypatch.setattr(nhip, "_scratch", spy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(side)
    torch.cuda.current_stream().wait_stream(side)
    assert places == ([side.cuda_stream] if scratch else [])
    for g, w in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
        assert owner(g) == side.cuda_stream
        assert torch.equal(g, w)


def test_results_freed_while_read():
    """A result dropped while the current stream still reads it is not handed out again by the other one."""
    x = torch.randn((4, 3000, 256), device="cuda")
    norm = nhip.GroupNorm(8, 256)
    want = norm.forward(x)
    nothing, big = torch.zeros_like(x), torch.randn((2048, 2048), device="cuda")
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    for _ in range(5):
        y = norm.forward(x, stream=side)
        main.wait_stream(side)
        for _ in range(20):
            big @ big  # the current stream is behind
        kept = y.clone()
        del y
        other = norm.forward(nothing, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(kept, want) and (other == 0).all()
