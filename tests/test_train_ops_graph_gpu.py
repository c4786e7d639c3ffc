"""The norms around a block, the checkpoints and the loss head in a captured HIP
graph: replayed on changing inputs, with eager calls between, every replay bit for
bit the eager result."""
import pytest
import torch

from aethelstream_amd import checkpoint, loss, norm

pytestmark = pytest.mark.gpu


def _randn(shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("m", [5, 300])
def test_captured_step_replays(m):
    d, v = 1024, 3000
    inputs = dict(h=_randn((m, d), 1, torch.bfloat16), res=_randn((m, d), 2),
                  dres=_randn((m, d), 3), targets=torch.zeros(m, dtype=torch.int64, device="cuda"))
    w, gate = 1 + 0.1 * _randn((d,), 4), _randn((d,), 5)
    head = (_randn((v, d), 6) * d ** -0.5).to(torch.bfloat16)
    dloss = torch.full((m,), 1.0 / m, device="cuda")

    def run():
        f = norm.block_norm_fwd(inputs["h"], inputs["res"], w, w, gate, 0.5)
        c = checkpoint.encode(f.res)
        out, lse = loss.linear_cross_entropy(f.y, head, inputs["targets"])
        dy, dhead = loss.linear_cross_entropy_bwd(f.y, head, inputs["targets"], lse, dloss)
        x, y, rms = checkpoint.decode_norm(c, w)
        b = norm.block_norm_bwd(dy, inputs["dres"], c, rms, w, inputs["h"], f.rms_post, w, gate,
                                0.5)
        return [f.res, f.y, c.codes, c.scales, out, lse, dy, dhead, x, y, rms, b.dres, b.dh,
                b.dw_pre, b.dw_post, b.dgate]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for replay in range(4):
        for i, name in enumerate(("h", "res", "dres")):
            t = inputs[name]
            t.copy_(_randn(t.shape, 10 * replay + i + 20, t.dtype))
        inputs["targets"].copy_(torch.arange(m, device="cuda") * (replay + 1) % v)
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
