"""The tcgen05 kernel of the 4-bit products, step by step.

It rounds a weight to fp16 under a power of two per row (the largest 15 |s| + |m| of the
row in 2^14..2^15) and sums in fp32.  Against 64-bit products of the weights so rounded
what is left is the sums' error: a step of 16 columns adds them to the accumulator, good
to 2^-22 of the accumulator and of the step's |x w| (fp32 has 2^-24; the tensor cores
align the terms and cut them).  With A the largest partial sum at the end of any 64
columns, a partial sum of any stretch is below 2 A and what its last 64 columns hold, so
that k / 16 steps come to 2^-22 (k / 16 * 2 A + 5 sum |x w|): a step of 64 columns left
out, or taken twice, is far outside."""
import pytest
import torch

from llama_pure_compute_b200 import _lib
from llama_pure_compute_b200.int4_linear import Int4Weight, int4_linear
from oracle.int4_ref import weight_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0, "a kernel flagged a device-side error"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def two_to(e):
    """2^e in 64 bits, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def to_half(x):
    """x (64 bits) rounded once to fp16's values, halves to even."""
    step = two_to(torch.frexp(x.abs().clamp(min=2.0 ** -14)).exponent - 11)
    return torch.round(x / step) * step


def rounded_weight(codes, s, m):
    """The weights that the kernel multiplies, in 64 bits."""
    top = (15 * s.double().abs() + m.double().abs()).amax(-1, keepdim=True)
    up = torch.where(top > 0, two_to(15 - torch.frexp(top).exponent), torch.ones_like(top))
    sh, mh = to_half(s.double() * up), to_half(m.double() * up)
    return to_half(weight_ref(codes, sh, mh)) / up


def random_weight(g, rows, k, group, dtype):
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    s = (torch.rand(rows, k // group, device=DEV, generator=g) + 0.5) * 0.004
    m = -7.5 * s * (torch.rand(rows, k // group, device=DEV, generator=g) * 0.4 + 0.8)
    return codes, s.to(dtype), m.to(dtype)


def sums_bar(x, w):
    """(x w^T, the bar above) in 64 bits, over 64 columns at a time."""
    T, k = x.shape
    z = torch.zeros(T, w.shape[0], dtype=torch.float64, device=DEV)
    top, size = torch.zeros_like(z), torch.zeros_like(z)
    for at in range(0, k, 64):
        xs, ws = x[:, at:at + 64].double(), w[:, at:at + 64]
        z = z + xs @ ws.mT
        size += xs.abs() @ ws.abs().mT
        top = torch.maximum(top, z.abs())
    return z, 2.0 ** -22 * (k / 16 * 2 * top + 5 * size)


def check(y, x, w, epilogue="store", resid=None):
    z, e = sums_bar(x, w)
    if epilogue == "residual":
        z = z + resid.double()
        e = e + z.abs() * 2.0 ** -23
    if epilogue == "swiglu":
        n = z.shape[1] // 2
        gt, up, eg, eu = z[:, :n], z[:, n:], e[:, :n], e[:, n:]
        silu = gt * torch.sigmoid(gt)
        z = silu * up
        # silu' <= 1.1; the exponential and the division are good to 2^-20
        e = 1.1 * eg * (up.abs() + eu) + (silu.abs() + 1.1 * eg) * eu + z.abs() * 2.0 ** -20
    far = (y.double() - z).abs()
    bar = z.abs() * (torch.finfo(y.dtype).eps / 2) + e + torch.finfo(y.dtype).tiny * 2.0 ** -8
    assert (far <= bar).all(), (far / bar).max().item()


def make(g, n, k, group, dtype, epilogue):
    codes, s, m = random_weight(g, 2 * n if epilogue == "swiglu" else n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group,
                              layout="swiglu" if epilogue == "swiglu" else "linear")
    return w, rounded_weight(codes, s, m)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,n,k,group,epilogue", [
    (17, 1225, 16384, 128, "store"), (32, 301, 65536, 64, "residual"), (33, 601, 8192, 128, "swiglu"),
    (64, 65, 65536, 128, "swiglu"), (48, 3000, 4096, 32, "residual"), (64, 40000, 128, 128, "store"),
    (20, 12000, 1088, 32, "swiglu"), (64, 4096, 4096, 64, "store"),
    # few tokens whose x does not fit the other kernel's shared memory
    (2, 2700, 28672, 128, "store"), (4, 2700, 28672, 32, "residual"), (5, 1400, 28672, 64, "swiglu"),
    (8, 2700, 28672, 128, "residual"), (8, 3500, 11008, 128, "swiglu"), (7, 7000, 11008, 64, "store"),
    # 9 to 16 on large weights
    (9, 19000, 4096, 128, "store"), (16, 9600, 4096, 32, "swiglu")])
def test_every_step_counts_once(dtype, tokens, n, k, group, epilogue):
    g = gen(tokens + n + k)
    w, rounded = make(g, n, k, group, dtype, epilogue)
    assert (w.workspace_bytes(tokens) > 0) == (dtype == BF)  # the kernel meant
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    r = torch.randn(tokens, n, device=DEV, generator=g).to(dtype) if epilogue == "residual" else None
    y = int4_linear(x, w, epilogue, resid=r)
    check(y, x, rounded, epilogue, r)
    assert torch.equal(int4_linear(x, w, epilogue, resid=r), y)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k,group", [(2100, 4096, 128), (300, 32768, 32), (5000, 1088, 64)])
def test_single_columns(dtype, n, k, group):
    """One-hot tokens read the rounded weights one by one, exactly: the first and the last
    column of every 64, so that each step of each share of the columns is named."""
    g = gen(n)
    w, rounded = make(g, n, k, group, dtype, "store")
    cols = torch.arange(0, k, 64, device=DEV).repeat_interleave(2)
    cols[1::2] += 63
    for at in range(0, cols.numel(), 64):
        c = cols[at:at + 64]
        x = torch.zeros(64, k, dtype=dtype, device=DEV)
        x[torch.arange(c.numel(), device=DEV), c] = 1.0
        want = rounded[:, c].t().to(dtype)
        got = int4_linear(x, w)
        assert torch.equal(got[:c.numel()], want) and (got[c.numel():] == 0).all()


@pytest.mark.parametrize("dtype,ratio", [(BF, 2.0 ** -8), (BF, 2.0 ** -14), (BF, 2.0 ** -20), (HF, 2.0 ** -8),
                                         (HF, 2.0 ** -10)])
@pytest.mark.parametrize("tokens,n", [(17, 4500), (17, 5000), (64, 4500), (64, 5000)])
def test_groups_of_very_different_scale(dtype, ratio, tokens, n):
    """A token that lies on the groups of small scales sees those as exactly as any:
    2^-11 of each weight, whatever the row's other groups hold.  17 tokens on 4500 rows
    are another kernel's, which does not round them."""
    g = gen(tokens)
    k, group = 4096, 128
    rounds = (tokens, n) != (17, 4500)
    codes, s, m = random_weight(g, n, k, group, torch.float32)
    small = torch.arange(k // group, device=DEV) % 4 != 1
    lift = 16.0 if dtype == HF else 1.0  # keeps the small ones normal numbers
    s, m = ((t * lift * torch.where(small, ratio, 1.0)).to(dtype) for t in (s, m))
    w = Int4Weight.from_codes(codes, s, m, group_size=group)
    assert (w.workspace_bytes(tokens) > 0) == (dtype == BF and rounds)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    x[1::2] = torch.where(small.repeat_interleave(group), x[1::2], torch.zeros_like(x[1::2]))
    y = int4_linear(x, w)
    if rounds:
        check(y, x, rounded_weight(codes, s, m))
    exact = weight_ref(codes, s, m)
    z, e = sums_bar(x, exact)
    ax = x.double().abs() @ exact.abs().mT
    far = (y.double() - z).abs()
    bar = z.abs() * (torch.finfo(dtype).eps / 2) + e + ax * 2.0 ** -11 + torch.finfo(dtype).tiny * 2.0 ** -8
    assert (far <= bar).all(), (far / bar).max().item()


def test_extreme_rows():
    """Rows of zeros, of huge and of tiny weights: the row's power follows."""
    g = gen(9)
    n, k, group = 3000, 4096, 128
    codes, s, m = random_weight(g, n, k, group, torch.float32)
    size = torch.ones(n, 1, device=DEV)
    size[::5], size[1::5], size[2::5] = 2.0 ** 90, 2.0 ** -90, 0.0
    s, m = (s * size).to(BF), (m * size).to(BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=group)
    x = torch.randn(40, k, device=DEV, generator=g).to(BF)
    y = int4_linear(x, w)
    check(y, x, rounded_weight(codes, s, m))
    assert (y[:, 2::5] == 0).all() and y.isfinite().all()
