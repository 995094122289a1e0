"""Policy rows of calls that are several launches: rows on both sides of every launch's border, against 64 bits with the tolerances of
test_gpu_policy."""
import numpy as np
import pytest
import torch

from test_gpu_policy import U, close, exact, exact_grad

pytestmark = pytest.mark.gpu


def at_borders(rows, launch):
    """The call's first and last rows and those around the first row of every launch."""
    at = {0, 1, rows - 2, rows - 1}
    for r in range(launch, rows, launch):
        at |= {r - 2, r - 1, r, r + 1, min(r + 2, rows - 1)}
    return torch.tensor(sorted(at))


def check_rows(at, logits, actions, mask, temperature, top, out, up=None, grad=None):
    """Rows `at` of a call's outputs (and of its gradient, for the coefficients up)."""
    at = at.cuda()
    pick = lambda t: None if t is None else t[at]  # noqa: E731
    x, a = pick(logits), pick(actions)
    m = mask if mask is None or mask.dim() == 1 else pick(mask)
    e = exact(x, a, m, temperature, top)
    close(pick(out.log_z), e["log_z"], e["tol_z"], "log_z")
    close(pick(out.entropy), e["entropy"], e["tol_h"], "entropy")
    lp_tol = e["tol_z"] + 3 * U * np.where(np.isfinite(e["log_prob"]), np.abs(e["log_prob"]) + 2 * e["big"], 0)
    close(pick(out.log_prob), e["log_prob"], lp_tol, "log_prob")
    if top:
        assert np.array_equal(pick(out.top_action).cpu().numpy(), e["top_at"])
        t = e["tol_z"][:, None] + 3 * U * np.where(np.isfinite(e["top"]), np.abs(e["top"]) + 2 * e["big"][:, None], 0)
        close(pick(out.top_log_prob), e["top"], t, "top_log_prob")
    if grad is not None:
        close(pick(grad), *exact_grad(e, a, *(pick(u) for u in up), temperature, logits.dtype), "gradient")


def coefficients(rows, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(rows, generator=g, device="cuda") for _ in range(3)]


def test_long_call_of_wide_rows_is_cut_as_its_workspace_was_sized():
    """One row of 50 000 for 2^20 + 5: the five rows of the last launch alone would be cut, those of the call are not."""
    from muzero_amd.policy import policy_log_probs
    rows, n = 2 ** 20 + 5, 50000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, n, generator=g).to(torch.bfloat16).cuda()
    a = torch.randint(0, n, (rows,), generator=g).cuda()
    for top in (0, 3):
        out = policy_log_probs(x.expand(rows, n), a, top=top)
        check_rows(at_borders(rows, 2 ** 20), x.expand(rows, n), a, None, 1.0, top, out)
        assert bool((out.log_z == out.log_z[0]).all()) and bool((out.entropy == out.entropy[0]).all())
        del out


@pytest.mark.parametrize("n", [3, 8, 9, 20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_narrow_rows_than_a_launch_takes(n, dtype):
    """2^24 + 5 rows, with masks, actions, coefficients and alternatives of their own."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    rows, top = 2 ** 24 + 5, 2
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    a = torch.randint(-1, n, (rows,), generator=g, device="cuda")
    m = torch.rand(rows, n, generator=g, device="cuda") < 0.8
    up = coefficients(rows, n)
    at = at_borders(rows, 2 ** 24)
    out = policy_log_probs(x, a, mask=m, temperature=0.7, top=top)
    check_rows(at, x, a, m, 0.7, top, out)
    for top in (0, 2):
        out, grad = policy_log_probs_grad(x, a, *up, mask=m, temperature=0.7, top=top)
        check_rows(at, x, a, m, 0.7, top, out, up, grad)
        del out, grad
    # every row: the parts between the borders are one launch's
    values = policy_log_probs(x, a, mask=m, temperature=0.7)
    z = (x.float() / 0.7).masked_fill(~m, -torch.inf)
    want = torch.logsumexp(z, 1)
    # products, differences, exponentials and sums of both sides: 64 roundings of terms of at most |z| + log n
    tol = 64 * U * (1 + z.masked_fill(~m, 0.0).abs().amax(1) + np.log(n))
    assert bool(((values.log_z == want) | ((values.log_z - want).abs() <= tol)).all())


@pytest.mark.parametrize("n", [2049, 4100, 8195])
def test_more_wide_rows_than_a_launch_takes(n):
    """2^20 + 5 rows that a wave holds (up to 8192), and that a block walks: one row of logits for all, actions and coefficients of their own,
    gradients of every row."""
    from muzero_amd.policy import policy_log_probs_grad
    rows = 2 ** 20 + 5
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, n, generator=g).half().cuda().expand(rows, n)
    m = (torch.rand(n, generator=g) < 0.8).cuda()
    a = torch.randint(-1, n, (rows,), generator=g).cuda()
    up = coefficients(rows, n)
    for top in (0, 2):
        out, grad = policy_log_probs_grad(x, a, *up, mask=m, temperature=1.3, top=top)
        check_rows(at_borders(rows, 2 ** 20), x, a, m, 1.3, top, out, up, grad)
        assert bool((out.log_z == out.log_z[0]).all())
        del out, grad


def test_a_block_a_row_for_more_rows_than_blocks_of_a_launch():
    """2^24 + 5 rows of 2049: a wave could hold them, their alternatives are looked for by a block each."""
    from muzero_amd.policy import policy_log_probs
    rows, n = 2 ** 24 + 5, 2049
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, n, generator=g).half().cuda().expand(rows, n)
    a = torch.randint(-1, n, (rows,), generator=g).cuda()
    out = policy_log_probs(x, a, top=1)
    check_rows(torch.cat([at_borders(rows, 2 ** 20), at_borders(rows, 2 ** 24)]), x, a, None, 1.0, 1, out)
    assert bool((out.log_z == out.log_z[0]).all()) and bool((out.top_action == out.top_action[0]).all())


@pytest.mark.parametrize("n, odd", [(2 ** 28, 0), (2 ** 28 - 3, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_widest_row(n, odd, dtype):
    """2^28 logits, cut over 256 blocks of 256 threads: q = n / 65536 + 40 roundings one after the other in a sum, in the notation of
    test_gpu_policy; alternatives and the action near the row's end."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n + odd, generator=g, device="cuda").to(dtype)[odd:][None]
    best = torch.cat([torch.arange(n - 20, n), torch.tensor([0, 1, 2 ** 27, 2 ** 27 + 1]), torch.arange(2 ** 20, 2 ** 20 + 8)]).cuda()
    x[0, best] = 12.0 - torch.arange(32, device="cuda").to(dtype) / 8       # exact, apart from each other and from the rest
    a = torch.tensor([n - 2], device="cuda")
    up = [torch.full((1,), c, device="cuda") for c in (0.7, -0.3, 0.2)]
    out = policy_log_probs(x, a, top=32)
    both, grad = policy_log_probs_grad(x, a, *up)
    z = x[0].double()
    d = z - 12.0
    p = torch.exp(d)
    s = float(p.sum())
    p /= s
    D1, D2 = float((p * -d).sum()), float((p * d * d).sum())
    log_z, h = 12.0 + np.log(s), float(np.log(s)) + D1
    q = n / 65536 + 40
    for o in (out, both):
        assert abs(float(o.log_z) - log_z) <= q * U + 3 * U * D1 + 3 * U * 12
        assert abs(float(o.entropy) - h) <= (q + 4) * U * (1 + D1) + 3 * U * (D1 + D2)
        assert abs(float(o.log_prob) - float(z[n - 2] - log_z)) <= q * U + 3 * U * (D1 + 60)
    assert torch.equal(out.top_action[0].long(), best)
    logp = d - np.log(s)
    k = 0.2 - 0.7 + 0.3 * (logp + h)
    size = 0.9 + 0.3 * (logp.abs() + h)
    want = p * k
    tol = p * size * U * (q + 8 + 3 * (logp.abs() + 2 * D1 + 1)) + p * 0.3 * 2 * ((q + 4) * U * (1 + D1) + 3 * U * (D1 + D2 + 12))
    want[n - 2] += 0.7
    tol[n - 2] += 4 * U * 0.7
    tol += (want.abs() + tol) * torch.finfo(dtype).eps / 2 + 2.0 ** -125
    off = (grad[0].double() - want).abs()
    assert bool((off <= tol).all()), (int((off > tol).sum()), float((off / tol).max()))
