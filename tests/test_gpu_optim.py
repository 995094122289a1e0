"""Gradient norm and AdamW over many tensors on the GPU, against their definition.

Tolerances, u = 2^-24: m = b1 m + (1 - b1) g takes three roundings of terms that |b1 m| + |(1 - b1) g| bounds, and b1 itself is rounded once: 4 u of that; v
likewise with one more for the square.  The step lr_t m / (sqrt(v) r + eps) takes at most nine roundings besides those of m and v; w (1 - lr wd) two, the
difference one.  8-bit states: the codes follow from the 64-bit value and the 16 dither bits wherever the sum of both, in steps of the code,
stays away from a whole number by more than 64 u times the 16 steps that a code has at most, and by more than the value's own error in
steps (b1 m + (1 - b1) g may cancel: its error goes by its terms, not by what is left of them)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [1, 31, 32, 33, 64, 65, 0, 255, 4095, 4096, 4097, 10007, 3, 70001]


def make(sizes, dtype, seed, scale=0.1, odd=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = (torch.randn(n, generator=g) * scale * 10.0 ** (-(i % 4))).to(dtype)
        if odd:        # an odd start within an allocation
            whole = torch.zeros(n + 3, dtype=dtype, device="cuda")
            whole[3:] = t.cuda()
            out.append(whole[3:])
        else:
            out.append(t.cuda())
    return out


def mix(x):
    x &= 0xFFFFFFFF
    x ^= x >> 16
    x = x * 0xBB67AE85 & 0xFFFFFFFF
    x ^= x >> 15
    x = x * 0x6A09E667 & 0xFFFFFFFF
    return x ^ (x >> 16)


def dither(seed, step, at, n):
    key = mix((seed & 0xFFFFFFFF) ^ mix(step * 0x9E3779B9 + (seed >> 32)))
    r = mix((np.arange(at, at + n, dtype=np.int64) * 0x9E3779B1 + key) & 0xFFFFFFFF)
    return (r >> 16) / 65536.0, (r & 0xFFFF) / 65536.0


def blocks(x):
    return np.pad(x, (0, -len(x) % 32)).reshape(-1, 32)


def to_codes(x, r, tol):
    """(exponent bytes, values in units of the exponent, which are sure) by the definition, in float64."""
    b, r, tol = blocks(x), blocks(r), blocks(tol)
    most = np.abs(b).max(1)
    with np.errstate(divide="ignore"):
        e = np.where(most > 0, np.ceil(np.log2(np.where(most > 0, most, 1) / 448)), -127)
    e = np.where(most * 2.0 ** -e > 448, e + 1, e)
    e = np.where((most > 0) & (most * 2.0 ** (1 - e) <= 448), e - 1, e)
    e = np.maximum(e, -127)
    off = 64 * U + tol.max(1) / np.where(most > 0, most, 1)
    sure_e = (most == 0) | (np.abs(most * 2.0 ** -e / 448 - 1) > off) & (np.abs(most * 2.0 ** -e / 224 - 1) > off)
    y = np.abs(b) * 2.0 ** -e[:, None]
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(y, 1e-300))), -6) - 3)
    q = y / step + r
    sure = (np.abs(q - np.round(q)) > 64 * U * 16 + tol * 2.0 ** -e[:, None] / step) & sure_e[:, None]
    return (e + 127).astype(int), np.copysign(np.floor(q) * step, b), sure | (y == 0) & sure_e[:, None], step


class Oracle:
    """AdamW in float64 on the CPU, tensor by tensor."""

    def __init__(self, params, lr, betas, eps, wd, bits, master, max_norm, seed, step=0):
        self.w = [p.double().cpu().numpy() for p in params]
        self.m, self.v = ([np.zeros(len(w)) for w in self.w] for _ in range(2))
        self.lr, self.betas, self.eps, self.wd, self.bits, self.max_norm, self.seed, self.t = lr, betas, eps, wd, bits, max_norm, seed, step
        self.starts = np.cumsum([0] + [-(-len(w) // 64) * 64 for w in self.w])

    def step(self, grads):
        gs = [g.double().cpu().numpy() for g in grads]
        norm = math.sqrt(sum((g * g).sum() for g in gs))
        clip = min(1.0, self.max_norm / (norm + 1e-6)) if self.max_norm else 1.0
        self.t += 1
        (b1, b2), t = self.betas, self.t
        self.tol_m, self.tol_v, self.tol_w = [], [], []
        for i, g in enumerate(gs):
            g = g * clip
            self.tol_m.append(U * 4 * (np.abs(b1 * self.m[i]) + 2 * np.abs((1 - b1) * g)) + 2.0 ** -140)
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            self.tol_v.append(U * 8 * self.v[i] + 2.0 ** -126)
            size, den = self.lr / (1 - b1 ** t), np.sqrt(self.v[i]) / math.sqrt(1 - b2 ** t) + self.eps
            move = size * self.m[i] / den
            # sqrt of a v below the smallest normal number
            tol = size / den * self.tol_m[-1] + np.abs(move) * (16 * U + np.sqrt(2.0 ** -126) / den)
            new = self.w[i] * (1 - self.lr * self.wd) - move
            self.tol_w.append(tol + 3 * U * (np.abs(self.w[i]) + np.abs(new)))
            self.w[i] = new
        return norm


def near(x, y, tol, what):
    x = x.double().cpu().numpy()
    bad = ~(np.abs(x - y) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, first {x[bad][0]!r} for {y[bad][0]!r} +- {np.broadcast_to(tol, x.shape)[bad][0]:.3g}"


def flat(opt, name, i):
    return opt.state_tensors()[name][opt.starts[i]:opt.starts[i] + opt.counts[i]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("sizes", [[1], [5], [4096], [4097, 1], SIZES, [3] * 300, [1 << 22, 17]])
def test_norm(dtype, odd, sizes):
    from muzero_amd.optim import TensorList, grad_norm
    gs = make(sizes, dtype, len(sizes), odd=odd)
    want = math.sqrt(sum((g.double() ** 2).sum().item() for g in gs))
    got = grad_norm(gs)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(got.item() - want) <= U * want       # one rounding of an fp64 sum
    assert torch.equal(grad_norm(TensorList(gs)), got)
    assert abs(grad_norm(gs + [None], scale=-0.125).item() - want / 8) <= U * want / 8
    assert torch.equal(grad_norm(gs[0]), grad_norm([gs[0]]))


def test_norm_extremes():
    from muzero_amd.optim import grad_norm
    assert grad_norm(torch.zeros(70, device="cuda")).item() == 0.0
    assert grad_norm(torch.zeros(0, device="cuda")).item() == 0.0
    big = torch.full((1000,), 1e30, device="cuda")              # squares past fp32
    assert abs(grad_norm(big).item() / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    small = torch.full((1000,), 1e-30, device="cuda")
    assert abs(grad_norm(small).item() / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    big[3] = math.inf
    assert grad_norm(big).item() == math.inf
    big[4] = math.nan
    assert math.isnan(grad_norm(big).item())


@pytest.mark.parametrize("param", DTYPES)
@pytest.mark.parametrize("grad", DTYPES)
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("odd", [False, True])
def test_fp32_states(param, grad, master, odd):
    from muzero_amd.optim import AdamW
    if master and param is torch.float32:
        with pytest.raises(ValueError, match="master"):
            AdamW(make([3], param, 0), master_weights=True)
        return
    ps = make(SIZES, param, 1, scale=1.0, odd=odd)
    opt = AdamW(ps, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.1, max_grad_norm=0.5 if odd else None, master_weights=master)
    o = Oracle(ps, 3e-3, (0.9, 0.99), 1e-8, 0.1, 32, master, 0.5 if odd else 0.0, 0)
    for k in range(3):
        gs = make(SIZES, grad, 10 + k, odd=odd)
        norm = o.step(gs)
        opt.step(gs)
        if odd:
            assert abs(opt.grad_norm.item() - norm) <= 2 * U * norm
        for i, p in enumerate(ps):
            near(flat(opt, "exp_avg", i), o.m[i], o.tol_m[i] + (4 * U * np.abs(o.m[i])), f"m[{i}]")
            near(flat(opt, "exp_avg_sq", i), o.v[i], o.tol_v[i] * 2, f"v[{i}]")
            half = torch.finfo(param).eps / 2
            tiny = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}[param]
            if master:
                near(flat(opt, "master", i), o.w[i], o.tol_w[i], f"master[{i}]")
                near(p, o.w[i], o.tol_w[i] + half * np.abs(o.w[i]) * 1.01 + tiny, f"w[{i}]")
                o.w[i] = flat(opt, "master", i).double().cpu().numpy()
            else:
                near(p, o.w[i], o.tol_w[i] + (0 if param is torch.float32 else half * np.abs(o.w[i]) * 1.01 + tiny), f"w[{i}]")
                o.w[i] = p.double().cpu().numpy()
            o.m[i], o.v[i] = (flat(opt, s, i).double().cpu().numpy() for s in ("exp_avg", "exp_avg_sq"))
    assert opt.step_count == 3 and opt.skipped_count == 0


def test_against_torch():
    """The same rule as torch.optim.AdamW, over 20 steps in fp32."""
    from muzero_amd.optim import AdamW
    ps = make([40, 1000, 7], torch.float32, 1, scale=1.0)
    mine = [p.clone() for p in ps]
    theirs = [p.clone().requires_grad_(True) for p in ps]
    ref = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.05)
    opt = AdamW(mine, lr=1e-2, weight_decay=0.05)
    for k in range(20):
        gs = make([40, 1000, 7], torch.float32, 30 + k)
        for p, g in zip(theirs, gs):
            p.grad = g.clone()
        torch.nn.utils.clip_grad_norm_(theirs, 0.3)
        ref.step()
        opt.max_grad_norm = 0.3
        opt.step(gs)
    for p, q in zip(mine, theirs):
        # 20 steps of at most 1.1 lr each, every one off by 40 u of itself and w by 4 u
        assert (p - q).abs().max() <= 20 * (1.1e-2 * 40 * U + 4 * U * q.abs().max())


@pytest.mark.parametrize("param, master", [(torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("odd", [False, True])
def test_byte_states(param, master, odd):
    from muzero_amd.optim import AdamW
    grad = torch.float32 if odd else param
    seed = (7 << 32) + 11
    ps = make(SIZES, param, 2, scale=1.0, odd=odd)
    opt = AdamW(ps, lr=1e-3, weight_decay=0.01, state_bits=8, master_weights=master, seed=seed)
    o = Oracle(ps, 1e-3, (0.9, 0.999), 1e-8, 0.01, 8, master, 0.0, seed)
    sure_of, total = 0, 0
    for k in range(4):
        gs = make(SIZES, grad, 20 + k, odd=odd)
        for g in gs:
            g[::5] = 0.0        # weights that see no gradient
        o.step(gs)
        opt.step(gs)
        for i, p in enumerate(ps):
            n = opt.counts[i]
            if n == 0:
                continue
            r1, r2 = dither(seed, k + 1, opt.starts[i], n)
            root = np.sqrt(o.v[i])
            for name, x, r, tol in (("exp_avg", o.m[i], r1, o.tol_m[i]), ("exp_avg_root", root, r2, 8 * U * root + 2.0 ** -64)):
                e, y, sure, step = to_codes(x, r, tol)
                if name == "exp_avg_root":
                    y = np.where((y == 0) & (blocks(x) > 0), 2.0 ** -9, y)
                at = opt.starts[i] // 32
                got_e = opt.state_tensors()[name + "_exponent"].view(torch.uint8)[at:at + len(e)].cpu().numpy().astype(int)
                got = blocks(flat(opt, name, i).double().cpu().numpy())
                rows = sure.any(1)
                assert np.array_equal(got_e[rows], e[rows]), name
                assert np.array_equal(got[sure], y[sure]), name
                same = got_e == e
                assert (np.abs(got - y)[same] <= step[same]).all(), name      # unsure ones: the neighbour at most
                sure_of += int(sure[:, :].sum())
                total += sure.size
                value = (got * 2.0 ** (got_e[:, None] - 127)).reshape(-1)[:n]
                if name == "exp_avg":
                    o.m[i] = value
                else:
                    o.v[i] = value ** 2
            half = torch.finfo(param).eps / 2
            tiny = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}[param]
            rounded = 0 if param is torch.float32 else half * np.abs(o.w[i]) * 1.01 + tiny
            if master:
                near(flat(opt, "master", i), o.w[i], o.tol_w[i], "master")
            near(p, o.w[i], o.tol_w[i] + rounded, "w")
            o.w[i] = (flat(opt, "master", i) if master else p).double().cpu().numpy()
    assert sure_of > 0.99 * total


def test_byte_states_are_unbiased():
    """A second moment that one step moves by less than half a code: the dither moves the right share of the codes.  Share of n
    independent choices of probability q: within 6 sqrt(q (1 - q) / n)."""
    from muzero_amd.optim import AdamW
    n = 1 << 20
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], lr=0.0, state_bits=8, weight_decay=0.0, seed=5)
    s = opt.state_dict()
    s["step"] = 10
    s["exp_avg_root"] = torch.full((n,), 256.0).to(torch.float8_e4m3fn).cuda()
    s["exp_avg_root_exponent"] = torch.full((n // 32,), 119, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    opt.load_state_dict(s)
    g = torch.full((n,), 2.0, device="cuda")        # u = 1 -> sqrt(0.999 + 0.004), 0.384 of a step of 1/8 ... in units of 2^-8
    opt.step([g])
    u = math.sqrt(0.999 + 0.001 * 4)
    q = (u * 256 - 256) / 32
    up = (opt.state_tensors()["exp_avg_root"].float() == 288).double().mean().item()
    assert ((opt.state_tensors()["exp_avg_root"].float() == 256) | (opt.state_tensors()["exp_avg_root"].float() == 288)).all()
    assert abs(up - q) <= 6 * math.sqrt(q * (1 - q) / n)
    # the next step draws anew
    before = opt.state_tensors()["exp_avg_root"].clone()
    opt.load_state_dict({**s, "step": 11})
    opt.step([g])
    assert not torch.equal(before.view(torch.uint8), opt.state_tensors()["exp_avg_root"].view(torch.uint8))


def test_byte_states_extremes():
    """Blocks of zeros, one large value among tiny ones, denormals, infinities and NaN in one block alone."""
    from muzero_amd.optim import AdamW
    n = 6 * 32 + 5
    g = torch.zeros(n)
    g[32] = 1e10
    g[33:64] = 1e-10
    g[64:96] = 1e-38
    g[96] = math.inf
    g[128] = math.nan
    g[160:] = 1.0
    p = torch.ones(n, device="cuda")
    opt = AdamW([p], state_bits=8, weight_decay=0.0)
    opt.step([g.cuda()])
    m, u = (opt.state_tensors()[k].float() for k in ("exp_avg", "exp_avg_root"))
    e = opt.state_tensors()["exp_avg_exponent"].view(torch.uint8)
    assert (m[:32] == 0).all() and (u[:32] == 0).all() and (e[0] == 0) and (p[:32] == 1).all()
    assert (u[33:64] == 2.0 ** -9).all()            # never 0 under a root that is not
    assert e[3] == 255 and e[4] == 255 and torch.isnan(m[96:160]).all()
    assert (m[160:n] != 0).all() and e[5] == e[6] and torch.isfinite(p[160:]).all()
    assert (m[n:] == 0).all()
    opt.step([torch.ones(n, device="cuda")])
    assert torch.isnan(p[96:160]).all() and torch.isfinite(p[:96]).all() and torch.isfinite(p[160:]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_that_is_not_finite_skips_the_step(bits):
    from muzero_amd.optim import AdamW
    ps = make([100, 5000], torch.float32, 0, scale=1.0)
    opt = AdamW(ps, state_bits=bits, max_grad_norm=1.0)
    opt.step(make([100, 5000], torch.float32, 1))
    before = [p.clone() for p in ps], {k: v.clone() for k, v in opt.state_tensors().items()}
    for bad in (math.inf, math.nan):
        gs = make([100, 5000], torch.float32, 2)
        gs[1][4321] = bad
        opt.step(gs)
    assert all(torch.equal(p, q) for p, q in zip(ps, before[0]))
    assert all(torch.equal(v.view(torch.uint8), before[1][k].view(torch.uint8)) for k, v in opt.state_tensors().items())
    assert opt.step_count == 1 and opt.skipped_count == 2
    opt.step(make([100, 5000], torch.float32, 3))
    assert opt.step_count == 2 and not torch.equal(ps[0], before[0][0])


def test_parameters_without_gradient_stay():
    from muzero_amd.optim import AdamW
    ps = [p.requires_grad_(True) for p in make([50, 5000, 9], torch.float32, 0, scale=1.0)]
    opt = AdamW(ps, max_grad_norm=0.1)
    gs = make([50, 5000, 9], torch.float32, 1)
    ps[0].grad, ps[2].grad = gs[0], gs[2]
    keep = [p.detach().clone() for p in ps]
    opt.step()
    assert torch.equal(ps[1], keep[1]) and not torch.equal(ps[0], keep[0]) and not torch.equal(ps[2], keep[2])
    assert (flat(opt, "exp_avg", 1) == 0).all()
    assert abs(opt.grad_norm.item() - math.sqrt(sum((gs[i].double() ** 2).sum().item() for i in (0, 2)))) < 1e-6
    opt.zero_grad()
    with pytest.raises(ValueError, match="no parameter"):
        opt.step()


def test_storage_that_is_replaced_is_followed():
    from muzero_amd.optim import AdamW
    a, b = make([5000], torch.float32, 0), make([5000], torch.float32, 0)
    one, two = AdamW(a), AdamW(b)
    for k in range(3):
        g = make([5000], torch.float32, 5 + k)
        one.step(g)
        b[0].data = b[0].data.clone()
        two.step(g)
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_round_trip(bits):
    from muzero_amd.optim import AdamW
    ps = make(SIZES, torch.bfloat16, 0, scale=1.0)
    qs = [p.clone() for p in ps]
    one = AdamW(ps, state_bits=bits, master_weights=True, seed=9)
    for k in range(2):
        one.step(make(SIZES, torch.bfloat16, k))
    two = AdamW([q.copy_(p) for p, q in zip(ps, qs)], state_bits=bits, master_weights=True, seed=1)
    two.load_state_dict(one.state_dict())
    g = make(SIZES, torch.bfloat16, 7)
    one.step(g)
    two.step(g)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    with pytest.raises(ValueError, match="missing"):
        two.load_state_dict({"step": 1})
    bad = one.state_dict()
    bad["exp_avg"] = bad["exp_avg"][:-64]
    with pytest.raises(ValueError, match="exp_avg"):
        two.load_state_dict(bad)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("listed", [False, True])
def test_captured_step_replays_as_the_next_steps(bits, listed):
    from muzero_amd.optim import AdamW, TensorList
    sizes = [64 * 31, 5000, 2]
    a, b = make(sizes, torch.float32, 0, scale=1.0), make(sizes, torch.float32, 0, scale=1.0)
    gs = make(sizes, torch.float32, 1)
    lr = torch.tensor(1e-2, device="cuda")
    one = AdamW(a, lr=lr, state_bits=bits, max_grad_norm=0.2, seed=3)
    two = AdamW(b, lr=lr, state_bits=bits, max_grad_norm=0.2, seed=3)
    grads = TensorList(gs) if listed else gs
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step(grads)
    assert one.step_count == 0
    one.step(grads)             # eager before the first replay
    two.step(gs)
    for k in range(4):
        for g, h in zip(gs, make(sizes, torch.float32, 10 + k)):
            g.copy_(h)
        lr.fill_(1e-2 / (k + 1))
        graph.replay()
        two.step([g.clone() for g in gs])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        assert one.step_count == two.step_count == k + 2
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        gs[0].add_(0.0)
        with pytest.raises(ValueError, match="capture"):
            TensorList(gs)


def test_one_norm_for_two_optimizers_and_loss_scale():
    from muzero_amd.optim import AdamW, grad_norm
    a, b = make([1000], torch.float32, 0), make([300], torch.float32, 1)
    both = [t.clone() for t in a + b]
    ga, gb = make([1000], torch.float32, 2), make([300], torch.float32, 3)
    norm = grad_norm(ga + gb)
    for p, g in ((a, ga), (b, gb)):
        opt = AdamW(p, max_grad_norm=0.01)
        opt.step([t * 1024 for t in g], norm=norm, grad_scale=1 / 1024)
        assert torch.equal(opt.grad_norm, norm)
    AdamW(both, max_grad_norm=0.01).step(ga + gb)
    assert all(torch.equal(p, q) for p, q in zip(a + b, both))


@pytest.mark.parametrize("dtype, count, bits", [(torch.float32, 70_000_003, 32), (torch.bfloat16, 140_000_003, 32), (torch.float32, 70_000_003, 8)])
def test_long_lists_go_past_the_caches(dtype, count, bits):
    """Arrays of more than 256 MiB; two steps, the second from states that the first wrote.  8 bits: against the same step in two halves,
    each of them short enough to stay in the caches, and the first half (its dither counts from 0 as well) equal bit by bit."""
    from muzero_amd.optim import AdamW, grad_norm
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(count, generator=g, device="cuda").to(dtype)
    g1, g2 = (torch.randn(count, generator=g, device="cuda").mul_(0.01).to(dtype) for _ in range(2))
    norm = grad_norm([g1, w])
    want = float(torch.sqrt(sum((t.double() ** 2).sum() for t in (g1, w))))
    assert abs(float(norm) - want) <= 4 * U * want
    old = w.clone()
    opt = AdamW([w], lr=0.01, weight_decay=0.1, state_bits=bits, seed=3)
    opt.step([g1]), opt.step([g2])
    if bits == 8:
        half = 1 << 20
        part = old[:half].clone()
        other = AdamW([part], lr=0.01, weight_decay=0.1, state_bits=8, seed=3)
        other.step([g1[:half].contiguous()]), other.step([g2[:half].contiguous()])
        assert torch.equal(part, w[:half])
        for k, v in other.state_tensors().items():
            assert torch.equal(v.view(torch.uint8), opt.state_tensors()[k][:v.numel()].view(torch.uint8))
        assert not torch.equal(w[-1000:], old[-1000:])
        return
    m = v = 0
    x = old.double()
    del old
    for t, gr in ((1, g1.double()), (2, g2.double())):
        m, v = 0.9 * m + 0.1 * gr, 0.999 * v + 0.001 * gr * gr
        before = x
        x = x * (1 - 0.001) - 0.01 / (1 - 0.9 ** t) * m / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
        if dtype is not torch.float32:      # the first step's weight may round the other way where it lies next to a border
            rounded = x.to(dtype).double()
            x = rounded
    # each step's fp32 rounding: under 60 u lr and 2 u |w|; 2-byte weights round after each step, so the first one may differ by a step of theirs
    eps = torch.finfo(dtype).eps
    tol = 2 * (60 * U * 0.01 + 3 * U * x.abs()) + (2 * eps * torch.maximum(x.abs(), before.abs()) if dtype is not torch.float32 else 0.0)
    assert bool(((w.double() - x).abs() <= tol).all())


def test_saved_tensors_notice_the_step():
    from muzero_amd.optim import AdamW
    w = torch.ones(4, device="cuda", requires_grad=True)
    y = (w * w).sum()
    AdamW([w]).step([torch.ones(4, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_refusals():
    from muzero_amd.optim import AdamW, TensorList
    p = torch.zeros(10, device="cuda")
    for kw, word in ((dict(state_bits=16), "state_bits"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "eps"),
                     (dict(weight_decay=-1.0), "weight_decay"), (dict(max_grad_norm=0.0), "max_grad_norm")):
        with pytest.raises(ValueError, match=word):
            AdamW([p], **kw)
    for ps, word in (([p, p], "overlap"), ([p, p[3:5]], "overlap"), ([p.double()], "float64"), ([p, p.half()], "one type"),
                     ([torch.zeros(4, 4, device="cuda").t()[1:]], "contiguous")):
        with pytest.raises(ValueError, match=word):
            AdamW(ps)
    opt = AdamW([p])
    for g, word in (([p[:9]], "elements"), ([p, p], "2 gradients"), ([p.double()], "float64"), (TensorList([p[:9]]), "match")):
        with pytest.raises(ValueError, match=word):
            opt.step(g)
    with pytest.raises(ValueError, match="norm"):
        opt.step([torch.ones(10, device="cuda")], norm=torch.ones((), device="cuda"))
    assert opt.step_count == 0 and (p == 0).all()


def test_many_tensors_and_steps_on_a_side_stream():
    from muzero_amd.optim import AdamW, TensorList
    sizes = [(i * 37) % 300 for i in range(700)]
    a, b = make(sizes, torch.bfloat16, 0, scale=1.0), make(sizes, torch.bfloat16, 0, scale=1.0)
    one, two = AdamW(a, state_bits=8, max_grad_norm=1.0), AdamW(b, state_bits=8, max_grad_norm=1.0)
    gs = make(sizes, torch.bfloat16, 1)
    listed = TensorList(gs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            one.step(listed)
    s.synchronize()
    for _ in range(3):
        two.step(gs)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
def test_values_changed_between_steps_count(bits):
    """Each step against a new optimizer with those values that goes on from the same state."""
    from muzero_amd import _lib
    from muzero_amd.optim import AdamW
    sizes = [40, 5000]
    a = make(sizes, torch.float32, 0, scale=1.0)
    opt = AdamW(a, max_grad_norm=1.0, state_bits=bits)
    opt.step(make(sizes, torch.float32, 1))
    changes = (dict(betas=(0.5, 0.9)), dict(eps=1e-2), dict(weight_decay=0.5), dict(lr=0.1), dict(max_grad_norm=0.01), dict(seed=77),
               dict(max_grad_norm=None))
    values = dict(max_grad_norm=1.0)
    for k, change in enumerate(changes):
        values.update(change)
        b = [p.clone() for p in a]
        other = AdamW(b, state_bits=bits, **values)
        other.load_state_dict({n: v for n, v in opt.state_dict().items() if n != "seed"})
        before, g = [p.clone() for p in a], make(sizes, torch.float32, 2 + k)
        for name, v in change.items():
            setattr(opt, name, v)
        opt.step(g), other.step(g)
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and not torch.equal(a[0], before[0])
        for n, v in opt.state_tensors().items():
            assert torch.equal(v.view(torch.uint8), other.state_tensors()[n].view(torch.uint8))
    for name, bad in (("betas", (1.0, 0.9)), ("eps", -1.0), ("weight_decay", -0.1), ("lr", -1.0)):
        keep = getattr(opt, name)
        setattr(opt, name, bad)
        with pytest.raises(_lib.MzsError):
            opt.step(make(sizes, torch.float32, 1))
        setattr(opt, name, keep)
    assert opt.step_count == 1 + len(changes)


def test_an_optimizer_is_not_made_in_a_capture():
    from muzero_amd.optim import AdamW
    p = torch.ones(70, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="before the capture"):
            AdamW([p])
        p.mul_(2.0)
    graph.replay()
    assert bool((p == 2.0).all())       # the capture went on


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_waits_for_the_stream_that_made_the_optimizer(bits):
    """States, master weights and table are written on a stream that is busy; the first step runs on another one at once."""
    from muzero_amd.optim import AdamW, TensorList, grad_norm
    sizes = [4096 * 30, 77]
    a, b = make(sizes, torch.bfloat16, 0, scale=1.0), make(sizes, torch.bfloat16, 0, scale=1.0)
    gs = make(sizes, torch.bfloat16, 1)
    want = AdamW(b, state_bits=bits, master_weights=True, max_grad_norm=0.5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)
        opt, listed = AdamW(a, state_bits=bits, master_weights=True, max_grad_norm=0.5), TensorList(gs)
        assert not s.query()
    opt.step(listed)
    norm = grad_norm(listed)
    want.step(gs)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(norm, want.grad_norm)


def test_memory_of_a_step_on_another_stream_is_marked_as_its(monkeypatch):
    """A replaced table, and the states of an optimizer that goes: not given out again before that stream is through."""
    from muzero_amd.optim import AdamW
    p = make([5000], torch.float32, 0)
    opt = AdamW(p, max_grad_norm=1.0)
    g = make([5000], torch.float32, 1)
    marked = []
    record = torch.Tensor.record_stream
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: (marked.append((t.data_ptr(), s.cuda_stream)), record(t, s))[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p[0].data = p[0].data.clone()
    opt.step(g)                                 # a table of the current stream
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step(g), opt.step(g)
    s.synchronize()
    mine = [opt.control, opt.grad_norm, opt._workspace, opt._params_table.memory, *opt.state_tensors().values()]
    assert sorted(marked) == sorted((t.data_ptr(), s.cuda_stream) for t in mine)


def test_a_graph_keeps_the_tables_that_it_reads():
    """A captured step, then the parameters' storage replaced, an eager step and the list of gradients gone: the graph goes on with the
    storage that it was captured on."""
    from muzero_amd.optim import AdamW, TensorList
    sizes = [5000, 300]
    p, q = make(sizes, torch.float32, 0), make(sizes, torch.float32, 0)
    gs = make(sizes, torch.float32, 1)
    opt, other = AdamW(p), AdamW(q)
    listed = TensorList(gs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(listed)
    tables = [opt._params_table.memory.data_ptr(), listed.table.memory.data_ptr()]
    size = opt._params_table.memory.numel()
    del listed
    old = [t.data for t in p]
    for t in p:
        t.data = t.data.clone()
    opt.step(gs)
    fill = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(400)]
    assert not {t.data_ptr() for t in fill} & set(tables)       # before the graph reads them
    other.step(gs)
    assert all(torch.equal(t, u) for t, u in zip(p, q))
    for _ in range(2):
        before = [t.clone() for t in p]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, u) for t, u in zip(p, before)) and not any(torch.equal(t, u) for t, u in zip(p, old))
    assert opt.step_count == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_past_32_bits(bits):
    """One tensor of 2^32 + 5000 elements, zeros but for parts on both sides of 2^31 and 2^32 and at its ends: each part as a short tensor's
    own step (8 bits: those whose elements' numbers are equal in 32 bits, which is what the dither takes of them)."""
    from muzero_amd.optim import AdamW, grad_norm
    n, part = 2 ** 32 + 5000, 5000
    starts = [0, 2 ** 31 - 2500, 2 ** 32 - 5000, 2 ** 32]
    w, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    ws, gs = make([part] * 4, torch.bfloat16, 1, scale=1.0), make([part] * 4, torch.bfloat16, 2)
    for at, a, b in zip(starts, ws, gs):
        w[at:at + part], g[at:at + part] = a, b
    norm = grad_norm([g])
    want = math.sqrt(sum((b.double() ** 2).sum().item() for b in gs))
    assert abs(float(norm) - want) <= 4 * U * want
    opt = AdamW([w], lr=0.01, state_bits=bits, max_grad_norm=0.5, seed=5)
    for _ in range(2):
        opt.step([g])
    state = opt.state_tensors()
    for at, a, b in zip(starts, ws, gs):
        if bits == 8 and at % 2 ** 32:
            continue
        short = AdamW([a], lr=0.01, state_bits=bits, max_grad_norm=0.5, seed=5)
        for _ in range(2):
            short.step([b], norm=norm)
        assert torch.equal(w[at:at + part], a)
        for k, v in short.state_tensors().items():
            each = 32 if "exponent" in k else 1
            got = state[k].view(torch.uint8).view(v.dtype)[at // each:at // each + part // each]
            assert torch.equal(got.view(torch.uint8), v[:part // each].view(torch.uint8))
    quiet = w[2 ** 31 + 2500:2 ** 32 - 5000]
    assert not bool(quiet.any())
