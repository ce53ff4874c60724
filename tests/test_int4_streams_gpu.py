"""4-bit products beside the other kernels that hold tensor memory, each on a stream
of its own: everything finishes, with the results that each has alone."""
import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from llama_pure_compute_b200.int4_linear import Int4Weight, int4_linear
from llama_pure_compute_b200.packed_linear import PackedWeight, packed_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("other", ["pair", "packed 144", "packed 256", "packed 32"])
@pytest.mark.parametrize("tokens", [17, 32, 64])
def test_products_beside_other_clusters(tokens, other):
    g = torch.Generator(device=DEV).manual_seed(tokens)

    def rnd(*s):
        return (torch.randn(*s, device=DEV, generator=g) * 0.05).to(BF)
    w = Int4Weight(rnd(3000, 4096))
    x = rnd(tokens, 4096)
    if other == "pair":
        gate, up, nw, h = rnd(2048, 2048), rnd(2048, 2048), rnd(2048), rnd(512, 2048)
        beside = lambda: ops.rmsswiglu_forward(h, nw, gate, up, 1e-5)  # noqa: E731
    else:
        n = int(other.split()[1])
        pw, h = PackedWeight(rnd(1024, 4096)), rnd(n, 4096)
        beside = lambda: packed_linear(h, pw)  # noqa: E731
    calls = [lambda: int4_linear(x, w), beside]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for c, s, outs in zip(calls, streams, got):
            with torch.cuda.stream(s):
                outs.append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for outs, v in zip(got, want) for y in outs)
    assert _lib.device_status() == 0
