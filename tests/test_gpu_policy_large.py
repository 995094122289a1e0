"""Policy rows of large logits or low temperatures, where c = log2 e / T times the largest logit is past what fp32 counts in ones: masks
written as numbers, rows on both sides of the border (2^24) from which exponents are differences of logits.  Against 64 bits with the
tolerances of test_gpu_policy; where those follow |largest logit / T| and say nothing, against what equal logits have to give."""
import math

import numpy as np
import pytest
import torch

from test_gpu_policy import U, check, head

pytestmark = pytest.mark.gpu
WIDTHS = [3, 8, 9, 64, 300, 2048, 3000, 9000, 20000, 60001, 100001]     # every kernel, narrow to cut over blocks
TYPED = [(n, torch.float32) for n in WIDTHS] + [(n, torch.bfloat16) for n in WIDTHS if n not in (8, 300, 20000)]


def equal_rows(x, a, temperature, rows):
    """log-probability, entropy and gradient of rows whose logits are all alike."""
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    n = x.shape[1]
    g = torch.ones(x.shape[0], device="cuda")
    tol = (n / 64 + 24) * U * (1 + math.log(n))
    for out in (policy_log_probs(x, a, temperature=temperature), policy_log_probs_grad(x, a, g, temperature=temperature)[0]):
        for r in rows:
            assert abs(float(out.log_prob[r]) + math.log(n)) <= tol and abs(float(out.entropy[r]) - math.log(n)) <= tol
    _, grad = policy_log_probs_grad(x, a, g, temperature=temperature)
    for r in rows:
        want = np.full(n, -1.0 / n)
        want[int(a[r])] += 1.0
        off = np.abs(grad[r].double().cpu().numpy() * temperature - want)
        # 4 u of the action's own 1, then the rounding to the type
        assert np.all(off <= (tol + torch.finfo(x.dtype).eps) * (np.abs(want) + 1.0 / n) + 8 * U * (np.abs(want) > 0.5))


@pytest.mark.parametrize("n, dtype", TYPED)
@pytest.mark.parametrize("value", [-1e9, -5e9, -1e10, -1e12, -1e20, 1e10, 1e15, -3e37, 1.2e7, -1.2e7, 2e7, -2e7, 2.5e7, -2.5e7, 1e8])
def test_rows_of_large_logits(n, value, dtype):
    x, a, m = head(7, n, torch.float32, n)
    v = float(torch.tensor(value).to(dtype))
    step = abs(v) * torch.finfo(dtype).eps
    g = torch.Generator(device="cuda").manual_seed(n)
    x[0] = v
    x[1] = v + step * torch.randint(-3, 4, (n,), generator=g, device="cuda")                 # neighbours
    x[2, torch.rand(n, generator=g, device="cuda") < 0.5] = v                                # beside ordinary ones
    x[3], x[3, n // 2] = v, 0.0
    x[4] = v * (1.0 + torch.rand(n, generator=g, device="cuda"))                             # spread out
    x[5] = v
    m[0], m[3, 0], m[5, 0] = True, True, True
    x = x.to(dtype)
    check(x, a, None, 1.0, top=2)
    check(x, a, m, 1.0, top=0)
    equal_rows(x, a, 1.0, (0, 5))


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("border", [2.0 ** 24, -(2.0 ** 24), 2.0 ** 25, -(2.0 ** 25)])
def test_rows_at_the_border(n, border):
    """Logits one apart on both sides of the largest ones that exponents by one fma take: rows that end just below, at and just above it,
    whose parts lie on the other side."""
    at = round(border / math.log2(math.e))
    x, a, m = head(9, n, torch.float32, n + 1)
    g = torch.Generator(device="cuda").manual_seed(n)
    for r in range(9):
        top = at + 2 * (r - 4)
        x[r] = top - torch.randint(0, 12, (n,), generator=g, device="cuda")
        x[r, torch.randint(0, n, (1,), generator=g, device="cuda")] = top
    x[7] -= 40.0 * (torch.arange(n, device="cuda") // 64 % 2)
    m[:, 0] = True
    check(x, a, None, 1.0, top=1)
    check(x, a, m, 1.0, top=0)


@pytest.mark.parametrize("n, dtype", TYPED)
@pytest.mark.parametrize("temperature", [1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-30])
def test_low_temperatures(n, temperature, dtype):
    x, a, m = head(4, n, dtype, n)
    x[0], x[1] = 12.3, 7.1
    x[2] = (x[2] * 2).round() / 2       # ties share
    m[:, 0] = True
    check(x, a, m, temperature, top=1)
    check(x, a, None, temperature, top=0)
    equal_rows(x, a, temperature, (0, 1))


@pytest.mark.parametrize("n", WIDTHS)
def test_half_precision_past_the_border(n):
    """c l_i up to 9e7 with the largest fp16 numbers."""
    x, a, m = head(4, n, torch.float16, n)
    x[0], x[1], x[2] = 60000.0, -60000.0, 11.6
    x[3] = 65504.0 - 32.0 * torch.randint(0, 3, (n,), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda")
    m[:, 0] = True
    for temperature in (1e-3, 0.0051):
        check(x, a, m, temperature, top=1)
        check(x, a, None, temperature, top=0)
        equal_rows(x, a, temperature, (0, 1, 2))
