"""Gradients through the FLUX attention of a model with adapters, by every
attention backend that the framework calls."""
import pytest
import torch
from torch import nn
import torch.nn.functional as F
from torch.nn.attention import SDPBackend, sdpa_kernel

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2


class _Square(nn.Module):
    def __init__(self, d, g):
        super().__init__()
        self.out_features = d
        self.weight = nn.Parameter((torch.randn(d, d, generator=g, device="cuda") * d ** -0.5).to(torch.bfloat16))

    def forward(self, x, out=None):
        return F.linear(x, self.weight)


def _attention(heads, dim_head, seed):
    """An attention whose projections are plain bf16 linears."""
    from diffuser_b200 import flux
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = heads * dim_head
    att = flux.FluxAttention(d, heads, dim_head, added_kv=True).cuda()
    for name in ("to_q", "to_k", "to_v", "add_q_proj", "add_k_proj", "add_v_proj", "to_add_out"):
        setattr(att, name, _Square(d, g))
    att.to_out[0] = _Square(d, g)
    att = att.to(torch.bfloat16)
    att.differentiable = True
    return att


def _reference(att, x, ctx, dx, dc):
    """The same in 64 bits by the formula."""
    x, ctx = (t.detach().double().requires_grad_() for t in (x, ctx))
    h = att.heads
    lin = lambda m, t: t @ m.weight.detach().double().T  # noqa: E731
    split = lambda t: t.unflatten(-1, (h, -1)).transpose(1, 2)  # noqa: E731

    def rms(t, n):
        return t * (t.square().mean(-1, keepdim=True) + n.eps).rsqrt() * n.weight.detach().double()

    q = torch.cat([rms(split(lin(att.add_q_proj, ctx)), att.norm_added_q), rms(split(lin(att.to_q, x)), att.norm_q)], 2)
    k = torch.cat([rms(split(lin(att.add_k_proj, ctx)), att.norm_added_k), rms(split(lin(att.to_k, x)), att.norm_k)], 2)
    v = torch.cat([split(lin(att.add_v_proj, ctx)), split(lin(att.to_v, x))], 2)
    o = (torch.softmax(q @ k.transpose(-1, -2) / q.shape[-1] ** 0.5, -1) @ v).transpose(1, 2).flatten(2)
    n = ctx.shape[1]
    img, txt = lin(att.to_out[0], o[:, n:]), lin(att.to_add_out, o[:, :n])
    return (img, txt), torch.autograd.grad([img, txt], [x, ctx], [dx.double(), dc.double()])


BACKENDS = {"cudnn": (SDPBackend.CUDNN_ATTENTION, "Cudnn"), "flash": (SDPBackend.FLASH_ATTENTION, "Flash"),
            "efficient": (SDPBackend.EFFICIENT_ATTENTION, "Efficient")}


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("batch,heads,dim_head,s_img,s_txt", [(3, 4, 64, 35, 9), (1, 2, 128, 100, 33), (2, 3, 64, 1, 1)])
def test_attention_gradients(monkeypatch, backend, batch, heads, dim_head, s_img, s_txt):
    att = _attention(heads, dim_head, s_img)
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda s: torch.randn(batch, s, heads * dim_head, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, ctx, dx, dc = rn(s_img).requires_grad_(), rn(s_txt).requires_grad_(), rn(s_img), rn(s_txt)
    ran, plain = [], F.scaled_dot_product_attention

    def seen(*args, **kw):
        out = plain(*args, **kw)
        ran.append(out.grad_fn.name())
        return out

    monkeypatch.setattr(F, "scaled_dot_product_attention", seen)

    def step():
        with sdpa_kernel([BACKENDS[backend][0]]):
            out = att(x, ctx)
        return (*out, *torch.autograd.grad(out, [x, ctx], [dx, dc]))

    got = step()
    assert len(ran) == 1 and BACKENDS[backend][1] in ran[0], ran
    want, grads = _reference(att, x, ctx, dx, dc)
    # roundings one after another: projection, norm (4 ops), attention's weights
    # and result, output projection, and as many back: sqrt(8 / 3) H = 1.6 H
    # forward, sqrt(16 / 3) H = 2.3 H backward, twice that for the softmax's
    # condition at logits of a few units
    for i, (a, b) in enumerate(zip(got, (*want, *grads))):
        assert ((a.double() - b).norm() / b.norm()).item() <= (4 if i < 2 else 6) * H, i
    # captured and replayed, with no eager graph over the same leaves alive
    got = [t.detach() for t in got]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    for t in (dx, dc):
        t.mul_(-2)
    graph.replay()
    for i, (a, b) in enumerate(zip(again, got)):
        assert torch.equal(a, b if i < 2 else -2 * b) or ((a - (b if i < 2 else -2 * b)).norm() <= 4 * H * a.norm()), i
