"""Layer operators (nerf_loc_amd.layers) against their definitions in 64 bits.

Tolerances are worst-case bounds, element by element, computed in float64 beside each reference: e = 2^-24 is a float32
rounding, u a rounding to the tensor's type (half of torch.finfo(t).eps).  A sum of n products in float32, in any order,
is off by at most (n + 2) e times the sum of the products' magnitudes."""
import math

import pytest
import torch

from nerf_loc_amd import hip, layers

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ["none", "relu", "gelu", "silu"]
# |act'|, |act''| and the error of the kernel's own act and act' (beyond that of its argument), relative to 1 + |z|: the
# fitted tail is good to 1.3e-7 and the exponential's argument z^2 / 2 carries e z^2 into it
SLOPE, CURVE, ACT_ERR = 1.13, 0.8, 1.2e-6


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the spacing of the type's subnormal numbers."""
    f = torch.finfo(dt)
    return f.tiny * f.eps / 2


def act64(z, name):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def grad64(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def check(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    d = (got - want).abs()
    ok = (d <= bound) | torch.isnan(want) | (got == want)
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0])
        raise AssertionError("%s: %d of %d outside; first at %d: got %r, want %r, bound %r" % (
            what, int((~ok).sum()), ok.numel(), i, got.flatten()[i].item(), want.flatten()[i].item(),
            bound.expand_as(want).flatten()[i].item()))


class Layer:
    """The 64-bit values of a linear layer and the error bounds of its outputs and gradients."""

    def __init__(self, pieces, w, b, r, act, stored=True):
        self.x = torch.cat([p.detach().double() for p in pieces], -1)
        self.w = w.detach().double()
        self.act, dt = act, w.dtype
        self.dt, self.u, self.t = dt, half_step(dt), tiny(dt)
        K = self.w.shape[1]
        # bmm on contiguous operands only
        mag = self.x.abs() @ self.w.abs().t().contiguous()
        self.z = self.x @ self.w.t().contiguous()
        if b is not None:
            self.z = self.z + b.detach().double()
            mag = mag + b.detach().double().abs()
        self.ez = (K + 3) * E * mag
        self.y = act64(self.z, act)
        self.ey = SLOPE * self.ez + (0 if act in ("none", "relu") else ACT_ERR * (1 + self.z.abs()))
        if r is not None:
            self.y = self.y + r.detach().double()
            self.ey = self.ey + E * self.y.abs()
        self.ey = self.ey + self.u * (self.y.abs() + self.ey) + self.t

    def gradients(self, g):
        g = g.detach().double()
        gz = g * grad64(self.z, self.act)
        if self.act == "none":
            eg = torch.zeros_like(g)
        elif self.act == "relu":        # the sign of an argument within its error is open
            eg = g.abs() * (self.z.abs() <= self.ez + self.t)
        else:                           # the argument is stored rounded
            eg = g.abs() * (CURVE * (self.ez + self.u * self.z.abs() + self.t) + ACT_ERR * 4)
        M, N = g.shape
        eb = eg.sum(0) + (M + 4) * E * (gz.abs() + eg).sum(0)
        if self.act not in ("none", "relu"):
            eg = eg + self.u * (gz.abs() + eg) + self.t
        mag = gz.abs() + eg
        dx = gz @ self.w
        ex = eg @ self.w.abs() + (N + 2) * E * (mag @ self.w.abs())
        gzt, magt = gz.t().contiguous(), mag.t().contiguous()
        dw = gzt @ self.x
        ew = eg.t().contiguous() @ self.x.abs() + (M + 260) * E * (magt @ self.x.abs())
        db = gz.sum(0)
        out = lambda e, v: e + self.u * (v.abs() + e) + self.t
        return (dx, out(ex, dx)), (dw, out(ew, dw)), (db, out(eb, db))


def make(dev, dt, m, n, k, k2, bias, residual, seed, grad=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    new = lambda *s, scale=1.0: (torch.randn(*s, device=dev, generator=g) * scale).to(dt).requires_grad_(grad)
    x = [new(m, k)] + ([new(m, k2)] if k2 else [])
    return x, new(n, k + k2, scale=(k + k2) ** -0.5), new(n, scale=0.1) if bias else None, new(m, n) if residual else None, g


# one row to many, widths below, at and beside every tile; the last ones are aligned for the wide loads throughout
SIZES = [(1, 1, 1, 0), (1, 7, 5, 0), (1, 64, 300, 0), (2, 300, 17, 0), (3, 1024, 1024, 0), (16, 257, 129, 0), (17, 128, 2048, 0),
         (33, 5, 1000, 0), (65, 65, 65, 0), (130, 131, 63, 0), (257, 255, 511, 0), (1000, 4, 256, 0), (64, 256, 63, 256),
         (129, 128, 256, 27), (77, 40, 1, 1), (5, 33, 8, 1000), (300, 256, 64, 256), (128, 128, 128, 0), (256, 512, 320, 0),
         (1025, 640, 512, 0), (4096, 256, 256, 0), (2049, 264, 72, 8)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_and_gradients(dev, dtype, size):
    m, n, k, k2 = size
    dt = TYPES[dtype]
    i = SIZES.index(size)
    act, bias, residual = ACTS[i % 4], i % 3 != 1, i % 2 == 1
    x, w, b, r, g = make(dev, dt, m, n, k, k2, bias, residual, 100 + i, grad=True)
    y = layers.linear(x[0] if k2 == 0 else tuple(x), w, b, act, r)
    ref = Layer(x, w, b, r, act)
    check(y.detach(), ref.y, ref.ey, "y")
    gy = torch.randn(m, n, device=dev, generator=g).to(dt)
    leaves = x + [w] + ([b] if bias else []) + ([r] if residual else [])
    got = list(torch.autograd.grad(y, leaves, gy))
    (dx, ex), (dw, ew), (db, eb) = ref.gradients(gy)
    check(torch.cat(got[:len(x)], -1), dx, ex, "dx")
    check(got[len(x)], dw, ew, "dw")
    if bias:
        check(got[len(x) + 1], db, eb, "db")
    if residual:
        assert torch.equal(got[-1], gy)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_every_activation_with_and_without_its_neighbours(dev, dtype, act):
    dt = TYPES[dtype]
    for j, (bias, residual) in enumerate([(False, False), (True, False), (False, True), (True, True)]):
        x, w, b, r, g = make(dev, dt, 70, 72, 40, 0, bias, residual, 7 + j, grad=True)
        y = layers.linear(x[0], w, b, act, r)
        ref = Layer(x, w, b, r, act)
        check(y.detach(), ref.y, ref.ey, (act, bias, residual))
        gy = torch.randn(70, 72, device=dev, generator=g).to(dt)
        dx, dw = torch.autograd.grad(y, [x[0], w], gy)
        (rx, ex), (rw, ew), _ = ref.gradients(gy)
        check(dx, rx, ex, "dx")
        check(dw, rw, ew, "dw")


def test_linear_leading_dimensions_strides_and_views(dev):
    """Views into wider rows, transposed and broadcast operands: the same numbers as their contiguous copies."""
    g = torch.Generator(device=dev).manual_seed(3)
    big = torch.randn(6, 50, 131, device=dev, generator=g)
    w_big = torch.randn(90, 200, device=dev, generator=g)
    x, w = big[:, :, 3:66], w_big[5:77, 7:70]
    assert not x.is_contiguous() and not w.is_contiguous()
    y = layers.linear(x, w, activation="silu")
    assert tuple(y.shape) == (6, 50, 72)
    ref = layers.linear(x.contiguous(), w.contiguous(), activation="silu")
    assert torch.equal(y, ref)
    flat = big.reshape(300, 131)
    assert torch.equal(layers.linear(flat[:, 3:66], w, activation="silu"), ref.reshape(300, 72))
    wt = torch.randn(63, 72, device=dev, generator=g).t()
    assert torch.equal(layers.linear(x, wt), layers.linear(x.contiguous(), wt.contiguous()))
    row = torch.randn(1, 72, device=dev, generator=g)
    res = row.expand(300, 72)
    assert torch.equal(layers.linear(flat[:, 3:66], w, residual=res), layers.linear(flat[:, 3:66], w, residual=res.contiguous()))
    one = layers.linear(torch.randn(63, device=dev, generator=g), w)
    assert tuple(one.shape) == (72,)


def test_linear_broadcast_and_shared_leaves_get_their_gradients(dev):
    """One leaf in several places (both pieces, input and residual) and a gradient that is a broadcast scalar."""
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(40, 24, device=dev, generator=g, requires_grad=True)
    w = torch.randn(24, 48, device=dev, generator=g, requires_grad=True)
    y = layers.linear((x, x), w, None, "gelu", residual=x)
    y.sum().backward()
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    r = act64(torch.cat([x64, x64], -1) @ w64.t(), "gelu") + x64
    r.sum().backward()
    assert float((x.grad.double() - x64.grad).abs().max()) < 1e-4 and float((w.grad.double() - w64.grad).abs().max()) < 1e-4


def test_linear_gradients_against_differences(dev):
    """A directional derivative of a float32 layer by central differences of the 64-bit definition."""
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(20, 33, device=dev, generator=g, requires_grad=True)
    w = (torch.randn(17, 33, device=dev, generator=g) * 33 ** -0.5).requires_grad_()
    b = torch.randn(17, device=dev, generator=g, requires_grad=True)
    c = torch.randn(20, 17, device=dev, generator=g)
    for act in ("gelu", "silu"):
        grads = torch.autograd.grad((layers.linear(x, w, b, act) * c).sum(), [x, w, b])
        for t, dt_ in zip((x, w, b), grads):
            d = torch.randn(t.shape, device=dev, generator=g).double()
            f = lambda s: (act64((x.double() + (d * s if t is x else 0)) @ (w.double() + (d * s if t is w else 0)).t() +
                                 (b.double() + (d * s if t is b else 0)), act) * c.double()).sum()
            h = 1e-5
            want = float((f(h) - f(-h)) / (2 * h))
            assert abs(float((dt_.double() * d).sum()) - want) < 1e-4 * max(1.0, abs(want)), act


def test_second_derivatives_are_refused(dev):
    x = torch.randn(5, 8, device=dev, requires_grad=True)
    w = torch.randn(8, 8, device=dev, requires_grad=True)
    for y in (layers.linear(x, w, activation="silu"), layers.add_rms_norm(x, w[0])[0], layers.add_rms_norm(x, w[0], x)[0]):
        with pytest.raises(NotImplementedError, match="first derivatives"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_no_rows(dev, dtype):
    dt = TYPES[dtype]
    x = torch.empty(0, 9, dtype=dt, device=dev, requires_grad=True)
    w = torch.ones(5, 9, dtype=dt, device=dev, requires_grad=True)
    b = torch.ones(5, dtype=dt, device=dev, requires_grad=True)
    y = layers.linear(x, w, b, "relu")
    assert tuple(y.shape) == (0, 5)
    y.sum().backward()
    assert tuple(x.grad.shape) == (0, 9) and torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_non_finite_values_stay_in_their_rows(dev, dtype):
    """NaN and infinities reach the outputs that their row or column takes part in and no others (the zeros that pad a
    tile multiply nothing of a neighbour)."""
    dt = TYPES[dtype]
    for m, n, k in ((70, 40, 37), (200, 256, 128)):
        g = torch.Generator(device=dev).manual_seed(6)
        x = torch.randn(m, k, device=dev, generator=g).to(dt)
        w = torch.randn(n, k, device=dev, generator=g).to(dt)
        clean = layers.linear(x, w, activation="relu")
        bad = x.clone()
        bad[m - 1, k - 1] = float("nan")
        y = layers.linear(bad, w, activation="relu")
        assert bool(torch.isnan(y[m - 1]).all()) and torch.equal(y[:m - 1], clean[:m - 1])
        bad = x.clone()
        bad[3, 0] = float("inf")
        y = layers.linear(bad, w, activation="relu")
        assert torch.equal(y[3], torch.where(w[:, 0] > 0, float("inf"), 0.0).to(dt)) and torch.equal(y[4:], clean[4:])
        wide = torch.full((m, 2 * k), float("nan"), device=dev, dtype=dt)
        wide[:, :k] = x                         # NaN right behind every row
        assert torch.equal(layers.linear(wide[:, :k], w, activation="relu"), clean)


def test_linear_fp16_overflow_of_the_stored_argument(dev):
    """An argument beyond float16 is stored as an infinity; the derivatives there are 1 and 0, not NaN."""
    x = torch.tensor([[60000.0], [-60000.0]], dtype=torch.float16, device=dev, requires_grad=True)
    w = torch.tensor([[2.0]], dtype=torch.float16, device=dev)
    for act in ("gelu", "silu"):
        y = layers.linear(x, w, None, act)
        gx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert gx.flatten().tolist() == [2.0, 0.0]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_relu_keeps_what_its_zero_meets_out(dev, dtype):
    """An infinite or NaN gradient behind a closed ReLU reaches neither the inputs' nor the parameters' gradients: the
    gradient is the one of a zero there, bit for bit, whether y or the stored argument says what is closed."""
    dt = TYPES[dtype]
    for m, n, k in ((9, 12, 24), (300, 72, 40)):
        x, w, b, r, g = make(dev, dt, m, n, k, 0, True, True, 31)
        gy = torch.randn(m, n, device=dev, generator=g).to(dt)
        _, z = hip.linear(x[0], w, b, "relu", want_z=True)
        shut = z <= 0
        assert bool(shut.any()) and bool((~shut).any())
        for fill in (float("inf"), float("-inf"), float("nan")):
            for res in (None, r):
                got, want = [], []
                for out, fill_with in ((got, fill), (want, 0.0)):
                    leaves = [t.clone().requires_grad_() for t in (x[0], w, b)]
                    y = layers.linear(leaves[0], leaves[1], leaves[2], "relu", res)
                    out += torch.autograd.grad(y, leaves, torch.where(shut, torch.tensor(fill_with, device=dev, dtype=dt), gy))
                assert all(torch.equal(a, c) and bool(torch.isfinite(a).all()) for a, c in zip(got, want))


def test_linear_same_result_every_time_and_under_graph_replay(dev):
    """No atomics: repeated calls agree bit for bit; a captured forward and backward replays to the eager result with eager
    work in between."""
    x, w, b, r, g = make(dev, torch.bfloat16, 5000, 96, 80, 0, True, True, 21)
    gy = torch.randn(5000, 96, device=dev, generator=g).bfloat16()
    step = lambda: (lambda y, z: (y,) + hip.linear_backward(gy, x[0], w, z, "gelu"))(*hip.linear(x[0], w, b, "gelu", r, want_z=True))
    first = [t.clone() for t in step() if t is not None]
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, [t for t in step() if t is not None]))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        held = [t for t in step() if t is not None]
    for _ in range(3):
        for t in held:
            t.zero_()
        x[0].mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, [t for t in step() if t is not None]))
        torch.randn(1 << 16, device=dev).sum().item()


def test_linear_on_side_streams_at_once(dev):
    """Backward passes on two streams at once: each has scratch of its own."""
    sets = [make(dev, torch.float16, 20000, 136, 104, 0, True, False, 30 + i) for i in range(2)]
    gys = [torch.randn(20000, 136, device=dev, generator=s[4]).half() for s in sets]

    def step(s, gy):
        y, z = hip.linear(s[0][0], s[1], s[2], "silu", want_z=True)
        return hip.linear_backward(gy, s[0][0], s[1], z, "silu")
    want = [step(s, gy) for s, gy in zip(sets, gys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, s, gy in zip(streams, sets, gys):
            with torch.cuda.stream(st):
                got.append(step(s, gy))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)


def test_linear_offsets_beyond_32_bits(dev):
    """Row strides that take the last rows past 2^31 elements and 2^32 bytes."""
    rows, k = 70, 64
    store = torch.zeros(rows * (1 << 25) + k, dtype=torch.bfloat16, device=dev)      # 4.7 GB
    x = store.as_strided((rows, k), (1 << 25, 1))
    g = torch.Generator(device=dev).manual_seed(8)
    x.copy_(torch.randn(rows, k, device=dev, generator=g))
    w = torch.randn(32, k, device=dev, generator=g).bfloat16()
    c = x.contiguous()
    y, _ = hip.linear(x, w)
    assert torch.equal(y, hip.linear(c, w)[0])
    gy = torch.randn(rows, 32, device=dev, generator=g).bfloat16()
    assert torch.equal(hip.linear_backward(gy, x, w, want_x0=False, want_b=False)[2], hip.linear_backward(gy, c, w)[2])


def test_linear_result_over_its_residual(dev):
    """In the C interface y may be the residual itself: few rows, tiles, a cut product, and the streaming kernel."""
    lib = hip.lib()
    for m, n, k in ((5, 72, 64), (300, 200, 128), (73, 64, 4096), (131072, 256, 256), (65600, 64, 64)):
        g = torch.Generator(device=dev).manual_seed(m)
        x, w, r = (torch.randn(*s, device=dev, generator=g).bfloat16() for s in ((m, k), (n, k), (m, n)))
        want, _ = hip.linear(x, w, None, "silu", r)
        p = lambda t: t.data_ptr()
        need = lib.nerf_linear_workspace_bytes(1, p(x), k, k, None, 0, 0, p(w), k, m, n)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        assert lib.nerf_linear(1, p(x), k, k, None, 0, 0, p(w), k, None, 3, p(r), n, p(r), n, None, 0, m, n, p(ws), need,
                               torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(r, want), (m, n, k)


# the streaming kernels: every column and reduction group, partial last tiles, z kept or not
@pytest.mark.parametrize("size", [(131072 + 77, 256, 256), (131072, 200, 136), (65536 + 31, 256, 64), (65536, 136, 128), (65536 + 1, 64, 256),
                                  (65600, 8, 8), (65536, 104, 72), (70001, 128, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_streaming_kernels(dev, dtype, size):
    m, n, k = size
    dt = TYPES[dtype]
    for act, bias, residual in (("relu", True, False), ("gelu", False, True), ("silu", True, False), ("none", False, False)):
        x, w, b, r, g = make(dev, dt, m, n, k, 0, bias, residual, 700 + n, grad=True)
        y = layers.linear(x[0], w, b, act, r)
        ref = Layer(x, w, b, r, act)
        check(y.detach(), ref.y, ref.ey, ("y", act))
        gy = torch.randn(m, n, device=dev, generator=g).to(dt)
        dx, dw = torch.autograd.grad(y, [x[0], w], gy)
        (rx, ex), (rw, ew), _ = ref.gradients(gy)
        check(dx, rx, ex, ("dx", act))
        check(dw, rw, ew, ("dw", act))
        with torch.no_grad():
            assert torch.equal(layers.linear(x[0], w, b, act, r), y)


def test_linear_many_rows(dev):
    """More than 2^31 output elements: the last rows are where they belong."""
    m, n, k = (1 << 23) + 100, 264, 16
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(m, k, device=dev, generator=g).bfloat16()
    w = torch.randn(n, k, device=dev, generator=g).bfloat16()
    y = layers.linear(x, w, activation="relu")
    for lo in (0, m // 2, m - 300):
        assert torch.equal(y[lo:lo + 300], layers.linear(x[lo:lo + 300], w, activation="relu"))


# ---------------------------------------------------------------------------------------------------- norm
def norm64(x, w, r, eps):
    h = x.detach().double() + (0 if r is None else r.detach().double())
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, rstd, h * rstd * w.detach().double()


NORM_SIZES = [(1, 1), (1, 31), (5, 32), (300, 33), (64, 128), (67, 129), (3, 512), (130, 513), (9, 1024), (4099, 256), (6, 1025),
              (11, 2048), (4, 2055), (1, 4096), (7, 4100), (3, 8192), (2, 9001), (2, 16385), (2, 32768), (65, 7)]


@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_add_rms_norm_and_gradients(dev, dtype, size):
    m, n = size
    dt = TYPES[dtype]
    u, t = half_step(dt), tiny(dt)
    i = NORM_SIZES.index(size)
    g = torch.Generator(device=dev).manual_seed(200 + i)
    new = lambda *s, scale=1.0, at=0.0: (torch.randn(*s, device=dev, generator=g) * scale + at).to(dt).requires_grad_()
    x, w, r = new(m, n), new(n, scale=0.2, at=1.0), new(m, n, scale=2.0) if i % 3 else None
    eps = 1e-5
    y, h = layers.add_rms_norm(x, w, r, eps)
    rh, rstd, ry = norm64(x, w, r, eps)
    rr = (n / 2 + 8) * E
    check(h.detach(), rh, (E + u) * rh.abs() + t, "h")
    check(y.detach(), ry, ry.abs() * (rr + 5 * E + u) + t, "y")
    gy, gh = (torch.randn(m, n, device=dev, generator=g).to(dt) for _ in range(2))
    leaves = [x, w] + ([r] if r is not None else [])
    got = torch.autograd.grad([y, h], leaves, [gy, gh])
    hn, nn = rh * rstd, gy.double() * w.detach().double()
    dot = (nn * hn).mean(-1, keepdim=True)
    dx = gh.double() + rstd * (nn - hn * dot)
    eh = u + E + rr + 2 * E                               # relative error of hn: h stored rounded, rstd, the product
    edot = (nn.abs() * hn.abs()).mean(-1, keepdim=True) * (eh + (n + 6) * E)
    ex = rstd * (nn.abs() * (rr + 5 * E) + hn.abs() * (edot + (eh + 5 * E) * dot.abs())) + gh.double().abs() * 3 * E
    # without a residual the two parts meet in torch: each rounded once more
    ex = ex + (u * (dx.abs() + ex) + t) * (1 if r is not None else 2) + (0 if r is not None else u * (dx - gh.double()).abs())
    check(got[0], dx, ex, "dx")
    dw = (gy.double() * hn).sum(0)
    ew = (gy.double().abs() * hn.abs()).sum(0) * (eh + (m + 8) * E)
    check(got[1], dw, ew + u * (dw.abs() + ew) + t, "dw")
    if r is not None:
        assert torch.equal(got[0], got[2])


def test_add_rms_norm_more_rows_than_one_grid_dimension(dev):
    """More than 2^20 workgroups: the rows behind them are there."""
    m = (1 << 26) + 1000
    x = torch.full((m, 1), 3.0, dtype=torch.bfloat16, device=dev)
    x[-1] = -2.0
    y, _ = layers.add_rms_norm(x, torch.ones(1, dtype=torch.bfloat16, device=dev), eps=0.0)
    assert float(y[:-1].min()) == float(y[:-1].max()) == 1.0 and float(y[-1]) == -1.0


def test_add_rms_norm_of_zeros_and_non_finite_rows(dev):
    x = torch.zeros(4, 40, device=dev)
    w = torch.ones(40, device=dev)
    y, h = layers.add_rms_norm(x, w, x)
    assert torch.equal(y, x) and torch.equal(h, x)
    x[1, 3] = float("nan")
    x[2, 39] = float("inf")
    x[3] = 1.0
    y, _ = layers.add_rms_norm(x, w)
    assert bool(torch.isnan(y[1]).all()) and bool((y[0] == 0).all()) and float((y[3] - 1).abs().max()) < 1e-5
    assert bool(torch.isnan(y[2, 39])) and bool((y[2, :39] == 0).all())
    q, s, _ = layers.add_rms_norm_q8(x, w)
    v = q.float() * s[:, None]
    assert bool((v[0] == 0).all()) and bool(torch.isnan(v[1]).all()) and bool(torch.isnan(v[2]).all())
    assert float((v[3] - 1).abs().max()) < 1e-5 and float(s[0]) == 2.0 ** -126


def test_add_rms_norm_one_output_used(dev):
    """Only y, or only h, enters the loss."""
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn(30, 70, device=dev, generator=g, requires_grad=True) for _ in range(2))
    w = torch.ones(70, device=dev, requires_grad=True)
    y, h = layers.add_rms_norm(x, w, r)
    gx, gw, gr = torch.autograd.grad(h, [x, w, r], torch.ones_like(h), retain_graph=True)
    assert bool((gx == 1).all()) and bool((gr == 1).all()) and bool((gw == 0).all())
    gx, gr = torch.autograd.grad(y, [x, r], torch.ones_like(y))
    hd = (x + r).detach().double().requires_grad_()
    want, = torch.autograd.grad((hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-6)).sum(), hd)
    assert torch.equal(gx, gr) and float((gx.double() - want).abs().max()) < 1e-5


def test_add_rms_norm_views_and_no_rows(dev):
    g = torch.Generator(device=dev).manual_seed(2)
    big = torch.randn(3, 20, 100, device=dev, generator=g)
    w = torch.rand(61, device=dev, generator=g)
    x, r = big[:, :, 7:68], big.flip(0)[:, :, 2:63]
    y, h = layers.add_rms_norm(x, w, r)
    y2, h2 = layers.add_rms_norm(x.contiguous(), w, r.contiguous())
    assert tuple(y.shape) == (3, 20, 61) and torch.equal(y, y2) and torch.equal(h, h2)
    e = torch.empty(0, 61, device=dev, requires_grad=True)
    wl = w.clone().requires_grad_()
    y, h = layers.add_rms_norm(e, wl, e)
    (y.sum() + h.sum()).backward()
    assert tuple(e.grad.shape) == (0, 61) and torch.equal(wl.grad, torch.zeros_like(w))
    q, s, _ = layers.add_rms_norm_q8(e.detach(), w)
    assert tuple(q.shape) == (0, 61) and tuple(s.shape) == (0,)


@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_add_rms_norm_q8(dev, dtype, size):
    m, n = size
    dt = TYPES[dtype]
    g = torch.Generator(device=dev).manual_seed(300 + NORM_SIZES.index(size))
    new = lambda *s, scale=1.0, at=0.0: (torch.randn(*s, device=dev, generator=g) * scale + at).to(dt)
    x, w, r = new(m, n), new(n, scale=0.2, at=1.0), new(m, n, scale=2.0)
    q, s, h = layers.add_rms_norm_q8(x, w, r)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and tuple(s.shape) == (m,)
    rh, _, ry = norm64(x, w, r, 1e-6)
    rel = (n / 2 + 14) * E
    want = (ry.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    check(s, want, want * (rel + 2 * E), "scale")
    check(h, rh, (E + half_step(dt)) * rh.abs() + tiny(dt), "h")
    # half a step of e4m3: 2^-4 of the value, 2^-10 below its smallest normal number
    step = torch.maximum(ry.abs() * 2.0 ** -4, 2.0 ** -10 * want[:, None])
    check(q.double() * s.double()[:, None], ry, step * (1 + 8 * rel) + ry.abs() * 2 * rel, "y")
    assert float(q.float().abs().amax(-1).min()) == 448.0


# ---------------------------------------------------------------------------------------------------- 8-bit linear
Q8_SIZES = [(1, 1, 1), (1, 4096, 1024), (3, 50, 16), (5, 256, 300), (17, 63, 129), (64, 128, 128), (130, 257, 511), (300, 512, 1024),
            (1024, 640, 256), (513, 33, 48)]


def q8_operands(dev, m, n, k, seed):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rows(r, c, scale):
        x = torch.randn(r, c, device=dev, generator=g) * scale
        s = (x.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
        return (x / s[:, None]).to(torch.float8_e4m3fn), s
    return rows(m, k, 1.0) + rows(n, k, k ** -0.5) + (g,)


def group_cut(x, w):
    """What the 8-bit matrix instruction may cut off: of every aligned group of eight products each loses less than 2^-13
    of the largest."""
    m, k = x.shape
    pad = -k % 8
    x, w = torch.nn.functional.pad(x, (0, pad)), torch.nn.functional.pad(w, (0, pad))
    cut = torch.zeros(m, w.shape[0], dtype=torch.float64, device=x.device)
    for i in range(0, k + pad, 8):
        cut += (x[:, None, i:i + 8] * w[None, :, i:i + 8]).abs().amax(-1)
    return cut * (7 * 2.0 ** -13)


@pytest.mark.parametrize("size", Q8_SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_q8(dev, dtype, size):
    m, n, k = size
    dt = TYPES[dtype]
    i = Q8_SIZES.index(size)
    act = ACTS[i % 4]
    xq, xs, wq, ws, g = q8_operands(dev, m, n, k, 400 + i)
    b = (torch.randn(n, device=dev, generator=g) * 0.1).to(dt) if i % 3 else None
    r = torch.randn(m, n, device=dev, generator=g).to(dt) if i % 2 else None
    y = layers.linear_q8(xq, xs, wq, ws, b, act, r, out_dtype=dt)
    assert y.dtype == dt
    X, W, S, T = xq.double(), wq.double(), xs.double()[:, None], ws.double()
    z = X @ W.t().contiguous() * S * T
    ez = (k + 6) * E * (X.abs() @ W.abs().t().contiguous()) * S * T
    if dt != torch.float32:
        ez = ez + group_cut(X, W) * S * T
    if b is not None:
        z = z + b.double()
        ez = ez + E * z.abs()
    want = act64(z, act)
    err = SLOPE * ez + (0 if act in ("none", "relu") else ACT_ERR * (1 + z.abs()))
    if r is not None:
        want = want + r.double()
        err = err + E * want.abs()
    check(y, want, err + half_step(dt) * (want.abs() + err) + tiny(dt), "y")


def test_linear_q8_views_every_number_and_no_rows(dev):
    """All 254 finite e4m3 numbers, exactly; strided operands; NaN; an empty batch; leading dimensions."""
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8, device=dev)
    v = codes.view(torch.float8_e4m3fn)
    eye = torch.eye(254, device=dev).to(torch.float8_e4m3fn)
    one = torch.ones(254, device=dev)
    x = torch.diag(v.float()).to(torch.float8_e4m3fn)
    for dt in TYPES.values():
        y = layers.linear_q8(x, one, eye, one, out_dtype=dt)
        assert torch.equal(y.float(), torch.diag(v.float()))
    xq, xs, wq, ws, g = q8_operands(dev, 96, 40, 77, 9)
    big = torch.zeros(96, 131, device=dev, dtype=torch.float8_e4m3fn).view(torch.uint8).fill_(0x7f).view(torch.float8_e4m3fn)
    big.view(torch.uint8)[:, 5:82] = xq.view(torch.uint8)
    want = layers.linear_q8(xq, xs, wq, ws, activation="silu")
    assert torch.equal(layers.linear_q8(big[:, 5:82], xs, wq, ws, activation="silu"), want)
    assert torch.equal(layers.linear_q8(xq.reshape(4, 24, 77), xs.reshape(4, 24), wq, ws, activation="silu"), want.reshape(4, 24, 40))
    bad = xq.clone()
    bad.view(torch.uint8)[95, 76] = 0x7f
    y = layers.linear_q8(bad, xs, wq, ws, activation="silu")
    assert bool(torch.isnan(y[95]).all()) and torch.equal(y[:95], want[:95])
    assert tuple(layers.linear_q8(xq[:0], xs[:0], wq, ws).shape) == (0, 40)


def test_quantised_block_as_it_is_used(dev):
    """Norm to 8 bits, 8-bit layer with the residual, next norm: against the same block on the quantised numbers in 64
    bits, and near the unquantised one."""
    g = torch.Generator(device=dev).manual_seed(11)
    x, r = (torch.randn(200, 320, device=dev, generator=g).bfloat16() for _ in range(2))
    w = (torch.randn(320, 320, device=dev, generator=g) * 320 ** -0.5)
    wn = torch.ones(320, device=dev, dtype=torch.bfloat16)
    wq, ws = layers.quantize_weight(w)
    q, s, h = layers.add_rms_norm_q8(x, wn, r)
    y = layers.linear_q8(q, s, wq, ws, activation="relu", residual=h)
    n2, h2 = layers.add_rms_norm(y, wn, h)
    X, W = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    z = X @ W.t().contiguous()
    ey = (330 * E) * (X.abs() @ W.abs().t().contiguous()) + group_cut(q.double(), wq.double()) * s.double()[:, None] * ws.double()
    want = torch.relu(z) + h.double()
    check(y, want, ey + half_step(torch.bfloat16) * (want.abs() + ey), "block")
    hh, _, nn = norm64(y, wn, h, 1e-6)
    check(n2, nn, nn.abs() * (175 * E + half_step(torch.bfloat16)) + 1e-30, "norm")
    full = torch.relu((norm64(x, wn, r, 1e-6)[2]) @ w.double().t().contiguous()) + h.double()
    # each factor is off by at most 2^-4 of itself, in effect independently: 2^-4 / sqrt 3 each, together below 2^-4
    assert float((y.double() - full).norm() / (full - h.double()).norm()) < 2.0 ** -4


# products that are cut along their reduction (few tiles, long sums) and whose unaligned operands are copied first
@pytest.mark.parametrize("size", [(73, 409, 1280, 16), (73, 100, 3000, 0), (700, 520, 1021, 0), (1100, 515, 331, 129), (90, 1000, 5, 0),
                                  (65, 64, 4096, 0), (520, 801, 63, 400), (200, 3, 2000, 0), (66, 2000, 17, 0)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_cut_and_copied(dev, dtype, size):
    m, n, k, k2 = size
    dt = TYPES[dtype]
    for j, act in enumerate(("gelu", "none")):
        x, w, b, r, g = make(dev, dt, m, n, k, k2, True, True, 500 + j, grad=True)
        y = layers.linear(x[0] if k2 == 0 else tuple(x), w, b, act, r)
        ref = Layer(x, w, b, r, act)
        check(y.detach(), ref.y, ref.ey, "y")
        gy = torch.randn(m, n, device=dev, generator=g).to(dt)
        got = list(torch.autograd.grad(y, x + [w, b], gy))
        (dx, ex), (dw, ew), (db, eb) = ref.gradients(gy)
        check(torch.cat(got[:len(x)], -1), dx, ex, "dx")
        check(got[len(x)], dw, ew, "dw")
        check(got[len(x) + 1], db, eb, "db")


def test_linear_q8_cut_and_copied(dev):
    for m, n, k in ((73, 100, 3000), (700, 520, 1021), (128, 64, 4096)):
        xq, xs, wq, ws, g = q8_operands(dev, m, n, k, 600 + m)
        X, W = xq.double(), wq.double()
        z = X @ W.t().contiguous() * xs.double()[:, None] * ws.double()
        ez = (k + 6) * E * (X.abs() @ W.abs().t().contiguous()) * xs.double()[:, None] * ws.double()
        check(layers.linear_q8(xq, xs, wq, ws, out_dtype=torch.float32), z, ez + E * z.abs(), "float32")
        ez = ez + group_cut(X, W) * xs.double()[:, None] * ws.double()
        check(layers.linear_q8(xq, xs, wq, ws), z, ez + half_step(torch.bfloat16) * (z.abs() + ez), "bf16")


# the input gradient formed together with the pass through the activation: both widths of its reduction, partial last tiles,
# the first, the second or both pieces wide enough for it, columns that end inside a group of the weights
@pytest.mark.parametrize("size", [(131072 + 45, 256, 256, 0), (131072, 72, 184, 0), (131072 + 1, 128, 200, 0), (140000, 136, 256, 0),
                                  (131103, 256, 63, 256), (131072, 200, 256, 136), (32768, 256, 8, 0), (32768 + 31, 248, 72, 0),
                                  (40001, 128, 128, 0)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_gradient_through_the_activation_and_the_input_at_once(dev, dtype, size):
    m, n, k, k2 = size
    dt = TYPES[dtype]
    for act, residual in (("relu", False), ("relu", True), ("gelu", False), ("silu", False)):
        x, w, b, r, g = make(dev, dt, m, n, k, k2, True, residual, 900 + n, grad=True)
        y = layers.linear(x[0] if k2 == 0 else tuple(x), w, b, act, r)
        gy = torch.randn(m, n, device=dev, generator=g).to(dt)
        got = torch.autograd.grad(y, x + [w, b], gy, retain_graph=True)
        (dx, ex), (dw, ew), (db, eb) = Layer(x, w, b, r, act).gradients(gy)
        check(torch.cat(got[:len(x)], -1), dx, ex, ("dx", act))
        check(got[-2], dw, ew, ("dw", act))
        check(got[-1], db, eb, ("db", act))
        again = torch.autograd.grad(y, x + [w, b], gy, retain_graph=True)
        assert all(torch.equal(a, c) for a, c in zip(got, again))
        # without the parameters' gradients, and from a gradient that lies in wider rows
        wide = torch.full((m, n + 24), float("nan"), device=dev, dtype=dt)
        wide[:, 8:8 + n] = gy
        alone = torch.autograd.grad(y, x[-1], wide[:, 8:8 + n])[0]
        assert torch.equal(alone, got[len(x) - 1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_relu_keeps_out_what_its_zero_meets_with_many_rows(dev, dtype):
    """The same on the streaming kernel: infinities and NaN behind closed ReLUs leave every gradient as zeros there do."""
    dt = TYPES[dtype]
    m, n, k = 32768 + 5, 136, 128
    x, w, b, _, g = make(dev, dt, m, n, k, 0, True, False, 32)
    gy = torch.randn(m, n, device=dev, generator=g).to(dt)
    y, _ = hip.linear(x[0], w, b, "relu")
    for fill in (float("inf"), float("nan")):
        got, want = (hip.linear_backward(torch.where(y <= 0, torch.tensor(v, device=dev, dtype=dt), gy), x[0], w, y, "relu") for v in (fill, 0.0))
        for i in (0, 2, 3):
            assert torch.equal(got[i], want[i]) and bool(torch.isfinite(got[i]).all()), (fill, i)


def test_linear_training_streams_in_two_graphs_at_once(dev):
    """Two captured backward passes of the streaming kernels, replayed on two streams at a time: each has its own scratch."""
    cases = []
    for seed in (41, 42):
        x, w, b, _, g = make(dev, torch.bfloat16, 40000, 256, 256, 0, True, False, seed)
        gy = torch.randn(40000, 256, device=dev, generator=g).bfloat16()
        y, z = hip.linear(x[0], w, b, "gelu", want_z=True)
        call = lambda x=x, w=w, z=z, gy=gy: [t for t in hip.linear_backward(gy, x[0], w, z, "gelu") if t is not None]
        want = call()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            held = call()
        cases.append((graph, side, held, want, gy, call))
    for k in range(3):
        for graph, side, held, want, gy, call in cases:
            for t in held:
                t.zero_()
        torch.cuda.synchronize()
        for graph, side, held, want, gy, call in cases:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, side, held, want, gy, call in cases:
            assert all(torch.equal(a, c) for a, c in zip(held, want)), k
            assert all(torch.equal(a, c) for a, c in zip(call(), want)), k
