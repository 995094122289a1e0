"""Policy rows on the GPU against their definition in 64 bits.

Tolerances.  u = 2^-24 (half a step of fp32).  d_i = c (l_i - max) has three roundings (c, difference, product) and the
exponential two more units, so e_i is off by a factor 1 + (3 |d_i| ln 2 + 2) u at most; a sum of n terms over at least 64
lanes adds at most n / 64 + 16 roundings one after the other.  With q = n / 64 + 20 and the exact moments D1 = E|d|, D2 = E d^2 of
a row (d in natural units):
    log s     q u + 3 u D1                          log_z     that + 3 u |max / T|      (scale, product, sum)
    entropy   (q + 4) u (1 + D1) + 3 u (D1 + D2)
    p_i       q u + 3 u (|d_i| + D1) relative
The gradient multiplies p_i with a coefficient of at most |g_z| + |g_a| + |g_h| (|log p_i| + H), whose own error is 8 u of that, adds g_a
at one place, and rounds once to its type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def exact(logits, actions, mask, temperature, top):
    """The definitions in float64 on the CPU, row by row in numpy; and the tolerances."""
    l = logits.detach().double().cpu().numpy()
    R, n = l.shape
    ok = np.ones((R, n), bool) if mask is None else np.broadcast_to(mask.cpu().numpy().astype(bool), (R, n))
    ok = ok & (l != -np.inf)
    out = {k: np.zeros(R) for k in ("log_prob", "entropy", "log_z", "tol_z", "tol_h", "big", "D1")}
    out["p"], out["logp"], out["ok"] = np.zeros((R, n)), np.full((R, n), -np.inf), ok
    out["top"], out["top_at"] = np.full((R, top), -np.inf), np.full((R, top), -1)
    q = n / 64 + 20
    for r in range(R):
        z = l[r][ok[r]] / temperature
        a = -1 if actions is None else int(actions[r])
        if z.size == 0:
            out["log_z"][r] = -np.inf
            out["log_prob"][r] = -np.inf if 0 <= a < n else np.nan if a >= n else 0.0
            continue
        big = z.max()
        with np.errstate(invalid="ignore", over="ignore"):
            d = z - big
            s = np.exp(d).sum()
            p = np.exp(d) / s
            logp = d - np.log(s)
        out["log_z"][r] = big + np.log(s)
        out["entropy"][r] = -(p[p > 0] * logp[p > 0]).sum() if np.isfinite(s) else np.nan
        out["p"][r, ok[r]], out["logp"][r, ok[r]] = p, logp
        if not np.isfinite(s):
            out["log_z"][r] = np.nan
        out["log_prob"][r] = np.nan if a >= n else 0.0 if a < 0 else out["logp"][r, a] if np.isfinite(s) else np.nan
        far = np.where(p > 0, np.abs(d), 0.0)
        D1, D2 = (p * far).sum(), (p * far * far).sum()
        out["big"][r], out["D1"][r] = abs(big), D1
        out["tol_z"][r] = q * U + 3 * U * D1 + 3 * U * abs(big)
        out["tol_h"][r] = (q + 4) * U * (1 + D1) + 3 * U * (D1 + D2)
        if top:
            v = np.where(ok[r], l[r], -np.inf)
            order = np.lexsort((np.arange(n), -np.where(np.isnan(v), np.inf, v), ~np.isnan(v)))[:top]
            order = order[ok[r][order]]
            out["top_at"][r, :len(order)], out["top"][r, :len(order)] = order, out["logp"][r, order]
    return out


def exact_grad(e, actions, g_a, g_h, g_z, temperature, dtype):
    """Gradient and its tolerance, in float64."""
    R, n = e["p"].shape
    zero = np.zeros(R)
    a = np.full(R, -1) if actions is None else actions.cpu().numpy()
    g_a, g_h, g_z = (zero if g is None else g.double().cpu().numpy() for g in (g_a, g_h, g_z))
    g_a = np.where(a < 0, 0.0, g_a)
    p, logp = e["p"], np.where(e["p"] > 0, e["logp"], 0.0)
    k = g_z[:, None] - g_a[:, None] - g_h[:, None] * (logp + e["entropy"][:, None])
    size = np.abs(g_z)[:, None] + np.abs(g_a)[:, None] + np.abs(g_h)[:, None] * (np.abs(logp) + e["entropy"][:, None])
    g = p * k
    q = n / 64 + 20
    tol = p * size * U * (q + 8 + 3 * (np.abs(logp) + 2 * e["D1"][:, None] + 1))
    tol += p * np.abs(g_h)[:, None] * (e["tol_h"][:, None] + e["tol_z"][:, None])
    for r in range(R):
        if 0 <= a[r] < n and e["ok"][r, a[r]]:
            g[r, a[r]] += g_a[r]
            tol[r, a[r]] += 4 * U * abs(g_a[r])
    g[~e["ok"]] = 0.0       # forbidden actions' elements, also in a row that a NaN or an infinity poisons
    g, tol = g / temperature, tol / temperature
    smallest = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    tol += (np.abs(g) + tol) * torch.finfo(dtype).eps / 2 + smallest
    # exponentials below the smallest normal number are flushed to 0
    return g, tol + 2.0 ** -125 * size / temperature


def close(x, y, tol, what):
    # a value past the largest fp32 number and half its step rounds to infinity (1 / 0.25 times the lowest one, for instance)
    y = np.where(np.abs(y) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, y), y)
    x = x.detach().double().cpu().numpy()
    same = (x == y) | (np.isnan(x) & np.isnan(y))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(x - y) <= tol))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off, first at {i}: {x[i]!r}, expected {y[i]!r} +- {np.broadcast_to(tol, x.shape)[i]:.3g}")


def check(logits, actions=None, mask=None, temperature=1.0, top=0, seed=0):
    """Forward, separate gradient (autograd) and the joined call, all against 64 bits."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    R, n = logits.shape
    e = exact(logits, actions, mask, temperature, top)
    g = torch.Generator().manual_seed(seed)
    dev = logits.device
    up = [torch.randn(R, generator=g).to(dev) for _ in range(3)]
    if actions is None:
        up[0] = None
    leaf = logits.detach().requires_grad_(True)
    out = policy_log_probs(leaf, actions, mask=mask, temperature=temperature, top=top)
    roots = [(o, u) for o, u in zip(out[:3], up) if u is not None]
    auto, = torch.autograd.grad([o for o, _ in roots], leaf, [u for _, u in roots])
    both, joined = policy_log_probs_grad(logits, actions, *up, mask=mask, temperature=temperature, top=top)
    plain = policy_log_probs(logits.detach(), actions, mask=mask, temperature=temperature, top=top)
    if top:         # with and without alternatives are two ways
        _, alone = policy_log_probs_grad(logits, actions, *up, mask=mask, temperature=temperature)
        close(alone, *exact_grad(e, actions, *up, temperature, logits.dtype), "gradient without alternatives")
    want, tol = exact_grad(e, actions, *up, temperature, logits.dtype)
    for name, o in (("forward", out), ("joined", both), ("no grad", plain)):
        close(o.log_z, e["log_z"], e["tol_z"], name + " log_z")
        close(o.entropy, e["entropy"], e["tol_h"], name + " entropy")
        lp_tol = e["tol_z"] + 3 * U * np.where(np.isfinite(e["log_prob"]), np.abs(e["log_prob"]) + 2 * e["big"], 0)
        close(o.log_prob, e["log_prob"], lp_tol, name + " log_prob")
        if top:
            assert o.top_action.dtype == torch.int32 and o.top_action.shape == (R, top)
            assert np.array_equal(o.top_action.cpu().numpy(), e["top_at"]), name + " top_action"
            t = e["tol_z"][:, None] + 3 * U * np.where(np.isfinite(e["top"]), np.abs(e["top"]) + 2 * e["big"][:, None], 0)
            close(o.top_log_prob, e["top"], t, name + " top_log_prob")
    assert auto.dtype == joined.dtype == logits.dtype
    close(auto, want, tol, "autograd")
    close(joined, want, tol, "joined gradient")
    return e


def head(R, n, dtype, seed, scale=2.0):
    """Logits as a head gives them, a few actions ahead of the rest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, n, generator=g) * scale
    x[torch.arange(R), torch.randint(0, n, (R,), generator=g)] += 6.0
    a = torch.randint(0, n, (R,), generator=g)
    m = torch.rand(R, n, generator=g) < 0.7
    return x.to(dtype).cuda(), a.cuda(), m.cuda()


SIZES = [(1, 1), (5, 1), (1, 2), (257, 2), (1000, 3), (77, 4), (3, 5), (64, 7), (130, 8), (33, 9), (65, 15), (9, 16), (9, 17), (70, 31),
         (13, 32), (21, 33), (5, 63), (66, 64), (7, 65), (3, 127), (6, 128), (3, 129), (5, 255), (2, 256), (3, 257), (2, 511), (4, 512),
         (3, 513), (2, 1000), (2, 1024), (3, 1025), (2, 2047), (2, 2049), (3, 4096), (2, 4097), (2, 5003), (3, 8192), (2, 8193), (2, 10000),
         (1, 16385), (2, 32768), (1, 40001), (1, 59049), (2, 65537), (1, 83521), (3, 83521), (1, 100000), (1, 131073), (1, 200001)]


@pytest.mark.parametrize("R, n", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes_and_types(R, n, dtype):
    x, a, m = head(R, n, dtype, n + R)
    i = (n + R) % 3
    check(x, a if i else a.to(torch.int32), (None, m, m[0].contiguous())[i], (1.0, 0.5, 1.7)[i], top=(0, 5, 20)[(n * 7 + R) % 3])


@pytest.mark.parametrize("n", [1, 2, 4, 16, 19, 64, 100, 1000, 3000, 20000, 70001])
@pytest.mark.parametrize("top", [1, 2, 8, 20, 31, 32])
def test_alternatives_with_ties_in_many_places(n, top):
    """Few distinct values: nearly every rank is decided by the lower index; and values that only just differ."""
    g = torch.Generator().manual_seed(n * 100 + top)
    x = torch.randint(-2, 3, (3, n), generator=g).float()
    x[1] = 0.0
    x[1, n // 2:] = -0.0
    x[2] = torch.arange(n) * 2.0 ** -18     # ascending: every element is a new largest one
    m = torch.rand(3, n, generator=g) < 0.9
    check(x.cuda(), None, m.cuda(), top=top)
    check(x.cuda().to(torch.bfloat16), None, None, top=top)


@pytest.mark.parametrize("n", [2, 16, 17, 64, 300, 2048, 5000, 40000, 90001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_allow_little_or_nothing(n, dtype):
    R = 9
    x, a, _ = head(R, n, dtype, n)
    m = torch.ones(R, n, dtype=torch.bool, device="cuda")
    m[0] = False                                                # nothing allowed
    m[1] = False
    m[1, n - 1] = True                                          # one allowed, the last
    x[2] = -math.inf                                            # all -inf
    x[3, 1:] = -math.inf                                        # one left
    x[4] = torch.finfo(dtype).min                               # masked by numbers, all of them: uniform
    x[5, : n // 2] = torch.finfo(dtype).min                     # masked by numbers
    m[6, a[6]] = False                                          # the action itself forbidden
    x[6, a[6]] = math.nan                                       # ... and not a number there
    m[7, : n // 2] = False
    x[7, : n // 2] = math.inf                                   # infinities in masked places
    a[8] = -1
    e = check(x, a, m, top=min(n, 4))
    assert e["log_z"][0] == -math.inf and e["log_prob"][6] == -math.inf
    check(x[:6], None, None, 0.25, top=3)


@pytest.mark.parametrize("n", [3, 50, 1000, 50000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number_and_infinity_poison_their_row_alone(n, dtype):
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    x, a, _ = head(4, n, dtype, n)
    x[1, n // 2], x[2, n - 1] = math.nan, math.inf
    a[3] = n                                                    # out of range
    one = torch.ones(4, device="cuda")
    out, g = policy_log_probs_grad(x, a, one, one, one, top=2)
    for t in (out.log_prob, out.entropy, out.log_z):
        assert torch.isnan(t[1:3]).all() and torch.isfinite(t[0])
    assert torch.isnan(out.log_prob[3]) and torch.isfinite(out.log_z[3]) and torch.isnan(g[3]).all()
    assert torch.isnan(g[1:3]).all() and torch.isfinite(g[0].float()).all()
    assert out.top_action[1, 0] == n // 2 and out.top_action[2, 0] == n - 1
    good = policy_log_probs(x[:1], a[:1], top=2)       # the same way (with alternatives): the same bits
    assert torch.equal(good.log_z, out.log_z[:1])


@pytest.mark.parametrize("n", [4, 37, 64, 1001, 30001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(n, dtype):
    """Rows apart by an odd pitch, from an odd start, one row for all, transposed, leading dimensions; masks alike."""
    from muzero_amd.policy import policy_log_probs
    R = 6
    flat = (torch.randn(R * (n + 7) + 3, generator=torch.Generator().manual_seed(n)) * 2).to(dtype).cuda()
    x = flat[3:].view(R, n + 7)[:, 2:n + 2]
    a = torch.arange(R, device="cuda") % n
    mm = (torch.rand(R * (n + 5) + 1, generator=torch.Generator().manual_seed(n + 1)) < 0.8).cuda()
    m = mm[1:].view(R, n + 5)[:, 3:n + 3]
    check(x, a, m, top=3)
    check(x[:1].expand(R, n), a, m)
    check(x, a, m[:1].expand(R, n))
    check(x[0].contiguous().view(n, 1).expand(n, R).t(), a)
    wide = x.contiguous().view(2, 3, n)
    got = policy_log_probs(wide, a.view(2, 3), mask=m.contiguous().view(2, 3, n), top=2)
    want = policy_log_probs(x.contiguous(), a, mask=m.contiguous(), top=2)
    for s, t in zip(got, want):
        assert torch.equal(s.reshape(t.shape), t)
    one = policy_log_probs(x[0], a[0], mask=m[0], top=2)
    assert one.log_prob.shape == () and torch.equal(one.log_prob, want.log_prob[0]) and torch.equal(one.top_action, want.top_action[0])


@pytest.mark.parametrize("n", [3, 64, 700, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_in_place_and_in_a_wider_buffer(n, dtype):
    from muzero_amd.policy import policy_log_probs_grad
    x, a, m = head(7, n, dtype, n)
    g = torch.randn(7, generator=torch.Generator().manual_seed(1)).cuda()
    _, want = policy_log_probs_grad(x, a, g, g, mask=m)
    wide = torch.full((9, n + 11), 7.0, dtype=dtype, device="cuda")
    out = wide[:7, 5:n + 5]
    _, got = policy_log_probs_grad(x, a, g, g, mask=m, out=out)
    assert got is out and torch.equal(out, want)
    assert (wide[7:] == 7).all() and (wide[:, :5] == 7).all() and (wide[:, n + 5:] == 7).all()
    policy_log_probs_grad(x, a, g, g, mask=m, out=x)
    assert torch.equal(x, want)


def test_gradient_beside_the_logits_and_overlapping_them():
    from muzero_amd.policy import policy_log_probs_grad
    x, a, _ = head(6, 40, torch.float32, 0)
    g = torch.ones(6, device="cuda")
    _, want = policy_log_probs_grad(x, a, g)
    buffer = torch.zeros(12, 100, device="cuda")
    for at, to in ((buffer[:6, :40], buffer[:6, 40:80]), (buffer[:6, 60:], buffer[:6, :40]), (buffer[:6, :40], buffer[6:, 3:43])):
        at.copy_(x)
        _, got = policy_log_probs_grad(at, a, g, out=to)
        assert torch.equal(got, want) and torch.equal(at, x)
    for at, to in ((buffer[:6, :40], buffer[:6, 39:79]), (buffer[:6, 60:], buffer[:6, 30:70]), (buffer[:6, :40], buffer[1:7, :40]),
                   (buffer[:6, 60:], buffer[1:7, 59:99]), (buffer.view(-1)[:240].view(6, 40), buffer[:6, :40])):
        with pytest.raises(ValueError):
            policy_log_probs_grad(at, a, g, out=to)


def test_saved_outputs_and_inputs_notice_a_change():
    from muzero_amd.policy import policy_log_probs
    x, a, m = head(6, 300, torch.float32, 0)
    leaf = x.clone().requires_grad_()
    for change in (lambda out: out.entropy.mul_(2), lambda out: a.zero_(), lambda out: m.fill_(True)):
        out = policy_log_probs(leaf, a, mask=m)
        loss = (out.log_prob + out.log_z).sum()
        with torch.no_grad():
            change(out)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


@pytest.mark.parametrize("R, n", [(256, 1025), (300, 2049), (257, 8193), (256, 20000), (260, 30011)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_wide_rows(R, n, dtype):
    """Enough rows that a row is one block's, with and without alternatives; some rows of every kind among them."""
    x, a, m = head(R, n, dtype, n)
    m[3] = False
    m[4] = False
    m[4, n - 1] = True
    x[5] = -math.inf
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).min
    x[8, n // 2] = math.nan
    x[9, 0] = math.inf
    m[10, : n // 2], x[10, : n // 2] = False, math.nan
    x[11] = 0.0
    a[12] = -1
    check(x, a, m, 0.5, top=7)
    check(x[11:], a[11:], None, top=32)


@pytest.mark.parametrize("R, n, dtype", [(4100, 2501, torch.bfloat16), (1500, 7001, torch.float32), (4096, 4096, torch.float16)])
def test_gradients_of_long_lists(R, n, dtype):
    x, a, m = head(R, n, dtype, R)
    check(x, a, m, 1.3)


def test_large_logits_keep_their_gradient():
    """log_z of logits around 10^4 has no bits left for the sum; the gradient is taken from the maximum and the sum instead."""
    for n in (5, 300, 20000):
        x, a, _ = head(3, n, torch.float32, n)
        check(x + 10000.0, a)
        check(x * 1e30, a)


def test_gradient_against_differences():
    from muzero_amd.policy import policy_log_probs
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 11, generator=g).cuda().requires_grad_(True)
    a, w = torch.tensor([2, 10, -1]).cuda(), torch.tensor([0.3, -1.2, 0.7]).cuda()

    def value(x):
        o = policy_log_probs(x, a, temperature=0.8)
        return (w * o.log_prob + 0.5 * o.entropy * w - 0.2 * o.log_z).double().sum()
    grad, = torch.autograd.grad(value(x), x)
    # central differences: step h = 2^-6 leaves h^2 / 6 of a third derivative below 20, and 2^-22 / h of rounding
    h, tol = 2.0 ** -6, 20 * 2.0 ** -12 / 6 + 2.0 ** -16
    with torch.no_grad():
        for r in range(3):
            for i in range(11):
                d = torch.zeros_like(x)
                d[r, i] = h
                assert abs((value(x + d) - value(x - d)).item() / (2 * h) - grad[r, i].item()) < tol


def test_refusals():
    from muzero_amd import _lib
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    x = torch.zeros(4, 6, device="cuda")
    a = torch.zeros(4, dtype=torch.int64, device="cuda")
    for kw, word in ((dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                     (dict(top=33), "top"), (dict(top=-1), "top"), (dict(actions=a.float()), "actions"), (dict(actions=a[:3]), "actions"),
                     (dict(actions=a.cpu()), "actions"), (dict(mask=torch.ones(4, 5, dtype=torch.bool, device="cuda")), "mask"),
                     (dict(mask=torch.ones(4, 6, device="cuda")), "mask"), (dict(mask=torch.ones(6, dtype=torch.bool)), "mask")):
        with pytest.raises(ValueError, match=word):
            policy_log_probs(x, **kw)
    with pytest.raises(ValueError, match="float64"):
        policy_log_probs(x.double())
    with pytest.raises(ValueError, match="0 actions"):
        policy_log_probs(x[:, :0])
    with pytest.raises(ValueError, match="grad_entropy"):
        policy_log_probs_grad(x, a, grad_entropy=torch.zeros(3, device="cuda"))
    for out in (x.half(), x[:, :5], x[:1].expand(4, 6), torch.zeros(6, 4, device="cuda").t()):
        with pytest.raises(ValueError, match="out"):
            policy_log_probs_grad(x, a, out=out)
    with pytest.raises(_lib.MzsError, match="GPU"):
        policy_log_probs(x.cpu())
    empty = policy_log_probs(x[:0], a[:0], top=2)
    assert empty.log_prob.shape == (0,) and empty.top_action.shape == (0, 2)
    leaf = x[:0].clone().requires_grad_(True)
    policy_log_probs(leaf, a[:0]).log_prob.sum().backward()
    assert leaf.grad.shape == (0, 6)


@pytest.mark.parametrize("R, n, dtype", [(1, 83521, torch.float16), (6, 64, torch.float32), (40, 3, torch.float32), (3, 20001, torch.bfloat16)])
def test_captured_and_replayed(R, n, dtype):
    """Forward and joined gradient in a graph, replayed on new inputs with eager work between; two graphs in turn."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    x, a, m = head(R, n, dtype, 5)
    g = torch.randn(R, device="cuda")
    other = x.clone()

    def work(x):
        out = policy_log_probs(x, a, mask=m, top=5)
        both, grad = policy_log_probs_grad(x, a, g, g, g, mask=m, top=2)
        return [*out, *both, grad]
    work(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in (x, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(t))
        graphs.append(graph)
    for k in range(4):
        fresh = [head(R, n, dtype, 10 + 2 * k + i)[0] for i in range(2)]
        x.copy_(fresh[0])
        other.copy_(fresh[1])
        want = [work(f) for f in fresh]
        for graph in graphs:
            graph.replay()
        eager = work(fresh[0])
        torch.cuda.synchronize()
        for o, w in zip(outs + [eager], want + [want[0]]):
            for s, t in zip(o, w):
                assert torch.equal(s, t)


def test_a_differentiable_call_is_not_captured():
    """Refused before anything is enqueued; the capture goes on, and eager graphs of the same leaves are as they were."""
    from muzero_amd.policy import policy_log_probs
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    a = torch.zeros(4, dtype=torch.int64, device="cuda")
    eager = policy_log_probs(x, a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="policy_log_probs_grad"):
            policy_log_probs(x, a)
        out = policy_log_probs(x.detach(), a)
    graph.replay()
    g, = torch.autograd.grad(eager.log_prob.sum(), x)
    assert torch.equal(out.log_prob, eager.log_prob.detach()) and torch.isfinite(g).all()


def test_side_stream_and_repeatability():
    from muzero_amd.policy import policy_log_probs_grad
    x, a, m = head(50, 5000, torch.bfloat16, 2)
    g = torch.randn(50, device="cuda")
    want = policy_log_probs_grad(x, a, g, g, mask=m, top=6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [policy_log_probs_grad(x, a, g, g, mask=m, top=6) for _ in range(3)]
    s.synchronize()
    for out, grad in got:
        assert torch.equal(grad, want[1])
        for p, q in zip(out, want[0]):
            assert p is None and q is None or torch.equal(p, q)


def test_many_short_rows():
    """More rows than a launch has blocks, and row offsets that pass 2^31 bytes."""
    from muzero_amd.policy import policy_log_probs
    R, n = 2 ** 20 + 3, 3
    x = torch.randn(R, n, device="cuda")
    a = torch.randint(0, n, (R,), device="cuda")
    out = policy_log_probs(x, a, top=1)
    z = x.double()
    lz = torch.logsumexp(z, 1)
    assert ((out.log_z.double() - lz).abs() <= 1e-6 * (1 + lz.abs())).all()
    assert torch.equal(out.top_action[:, 0].long(), x.argmax(1))
    R, n = 40000, 30001         # 4.8 GB of fp32
    x = torch.zeros(R, n, dtype=torch.float32, device="cuda")
    x[-1, -1], x[R // 2, 7] = 3.0, 2.0
    out = policy_log_probs(x, torch.full((R,), n - 1, device="cuda"), top=1)
    assert out.top_action[-1, 0] == n - 1 and out.top_action[R // 2, 0] == 7 and out.top_action[0, 0] == 0
    flat, one = math.log(n), math.log(n - 1 + math.exp(3.0))
    assert abs(out.log_z[0].item() - flat) < 1e-4 and abs(out.log_z[-1].item() - one) < 1e-4
    assert abs(out.log_prob[-1].item() - (3.0 - one)) < 1e-4


@pytest.mark.parametrize("n", [9, 10, 12, 13, 16, 17, 24, 25, 32, 33, 48, 64, 65, 96, 127, 128, 192, 200, 256, 384, 500, 512, 700, 768, 1000,
                               1024, 1025, 1300, 1536, 1537, 2000, 2047, 2048])
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_many_rows(n, dtype):
    """Enough rows that few lanes hold each: 96 rows with ties, forbidden and infinite places over and over, the last ones cut off."""
    R, top = 96, (1, 7, 32)[n % 3]
    x, a, m = head(R, n, dtype, n)
    x[:40] = (x[:40] * 2).round() / 2
    x[40], x[41, n // 2:], m[42] = -math.inf, -math.inf, False
    m[43:48] = True
    x[44] = torch.finfo(dtype).min
    x[45] = 0.0
    e = exact(x, a, m, 0.5, top)
    times = 131072 * 8 // (R * n) + 2
    rows = R * times - 5
    from muzero_amd.policy import policy_log_probs
    o = policy_log_probs(x.repeat(times, 1)[:rows], a.repeat(times)[:rows], mask=m.repeat(times, 1)[:rows], temperature=0.5, top=top)
    index = np.arange(rows) % R
    assert np.array_equal(o.top_action.cpu().numpy(), e["top_at"][index])
    t = e["tol_z"][:, None] + 3 * U * np.where(np.isfinite(e["top"]), np.abs(e["top"]) + 2 * e["big"][:, None], 0)
    close(o.top_log_prob, e["top"][index], t[index], "top_log_prob")
    close(o.log_z, e["log_z"][index], e["tol_z"][index], "log_z")
    close(o.entropy, e["entropy"][index], e["tol_h"][index], "entropy")


@pytest.mark.parametrize("R, n", [(1, 49151), (1, 49152), (3, 49153), (127, 49152), (128, 49152), (40, 60001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_on_both_sides_of_a_cut(R, n, dtype):
    x, a, m = head(R, n, dtype, n)
    if R > 2:
        m[1], x[2, n // 3:] = False, -math.inf
    check(x, a, m, 0.8, top=6)


def test_two_streams_at_once():
    """Calls that cut their rows have a workspace each."""
    from muzero_amd.policy import policy_log_probs
    sets = [head(5, 70001 + i, torch.bfloat16, i) for i in range(2)]
    want = [policy_log_probs(x, a, mask=m, top=9) for x, a, m in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (s, (x, a, m)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(policy_log_probs(x, a, mask=m, top=9))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(w, o))


def test_backward_twice_and_of_parts():
    from muzero_amd.policy import policy_log_probs
    x, a, m = head(7, 300, torch.float32, 1)
    leaf = x.clone().requires_grad_()
    out = policy_log_probs(leaf, a, mask=m, top=2)
    one, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
    two, = torch.autograd.grad(out.log_prob.sum(), leaf, retain_graph=True)
    again, = torch.autograd.grad(out.entropy.sum(), leaf)
    assert torch.equal(one, again) and not torch.equal(one, two)
    out = policy_log_probs(leaf, a, mask=m)
    graph, = torch.autograd.grad(out.log_z.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):                           # once differentiable: refused, not silently wrong
        graph.sum().backward()


@pytest.mark.parametrize("shape", [(6, 9), (2, 3, 9), (9,)])
def test_outputs_are_tensors_of_their_own(shape):
    """Operations in place that autograd records are taken by each, and change no other."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    x = torch.randn(shape, device="cuda")
    g = torch.ones(shape[:-1], device="cuda")
    for call in (lambda: policy_log_probs(x, top=2), lambda: policy_log_probs_grad(x, grad_entropy=g, top=2)[0]):
        want, out = call(), call()
        scale = torch.full((), 2.0, device="cuda", requires_grad=True)
        for i in (0, 1, 2, 3):
            out[i].mul_(scale)
            assert out[i].requires_grad and torch.equal(out[i].detach(), 2 * want[i])
            assert all(torch.equal(o.detach(), w) and not o.requires_grad for o, w in zip(out[i + 1:], want[i + 1:]))
        got, = torch.autograd.grad(sum(o.sum() for o in out[:4]), scale)
        assert torch.allclose(got, sum(w.sum() for w in want[:4]), rtol=1e-5, atol=0)


@pytest.mark.parametrize("places", [2, 3, 4, 6, 8, 12, 16, 20, 22, 24])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_block_on_both_sides_of_each_step(places, dtype):
    """Rows that fill so many vectors a thread of a block's 512, one logit fewer and one more (an odd start in every second row)."""
    full = 512 * places * (4 if dtype is torch.float32 else 8)
    for n in (full - 1, full, full + 1):
        x, a, m = head(3, n, dtype, n)
        a[0], a[1] = 0, n - 1
        m[:2, 0], m[:2, -1] = True, True
        check(x, a, m, 0.9, top=0)
