"""The linears' scratch on several streams and under captured graphs: partial
sums of a split sum, and a weight decoded to bf16 with its ready counters."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# tokens, outputs, features, forced splits
SIZES = {"split": (48, 640, 1088, 3), "decoded": (1100, 640, 1024, 0)}


def _linears(n, k, count, adapters=True):
    from diffuser_b200 import modules, ops
    out = []
    for i in range(count):
        g = torch.Generator(device="cuda").manual_seed(i)
        lin = modules.Ltx23Nf4Linear(n, k, bias=False).cuda()
        lin.set_nf4_weight(*ops.ltx23_nf4_quantize(torch.randn(n, k, generator=g, device="cuda")))
        if adapters:
            lin = modules.AdapterLinear(lin, 1, 8)
            with torch.no_grad():
                lin.down.copy_(torch.randn(1, 8, k, generator=g, device="cuda"))
                lin.up.copy_(torch.randn(1, 8, n, generator=g, device="cuda"))
            lin.selection = modules.AdapterSelection(torch.zeros(1, dtype=torch.int32, device="cuda"), 1)
        out.append(lin)
    return out


@pytest.fixture(params=SIZES)
def size(request):
    from diffuser_b200 import ops
    m, n, k, splits = SIZES[request.param]
    ops.set_tile_override(0, splits)
    plan = ops.plan_info(m, n, k)
    assert plan["splits"] == 3 if splits else plan["twophase"]
    assert ops.workspace_size(m, n, k) > 0
    yield m, n, k
    ops.set_tile_override(0, 0)


def test_two_streams_have_scratch_of_their_own(size):
    m, n, k = size
    mods = _linears(n, k, 2)
    xs = [torch.randn(m, k, device="cuda").to(torch.bfloat16) for _ in mods]
    with torch.no_grad():
        want = [lin(x) for lin, x in zip(mods, xs)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in mods], [[], []]
        for _ in range(30):
            for i, (lin, x, st) in enumerate(zip(mods, xs, streams)):
                with torch.cuda.stream(st):
                    got[i].append(lin(x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_a_captured_call_keeps_its_scratch(size):
    from diffuser_b200 import ops
    m, n, k = size
    lin, = _linears(n, k, 1, adapters=False)
    wider, = _linears(2 * n, 2 * k, 1, adapters=False)
    x = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    lin(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x)
    # an eager call that needs more, then everything that was given back taken
    wider(torch.randn(2 * m, 2 * k, device="cuda").to(torch.bfloat16))
    ops.release_workspaces()
    nbytes = ops.workspace_size(m, n, k)
    taken = [torch.full((nbytes,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    x.copy_(torch.randn(m, k, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, lin(x))
    assert all((t == 7).all() for t in taken) and ops.device_error() == 0
