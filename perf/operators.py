"""What is measured of the policy-head and optimizer operators: log-probabilities of given actions (with entropy, log
partition and the top alternatives), their gradient, the global gradient norm and the AdamW step.

Every operator has a plain form in elementary torch operations (`own` false) and the framework's call (`own` true).
Shapes: the self-play bench's 4096 slots, 500 moves a game, 2 .. 4 actions; the training batch of 128 samples x 5
unrolled steps; Box action spaces, whose actions are the cartesian product of `bins` samples per dimension (10 ** 5,
17 ** 4); parameter lists of the CartPole MLP and of generic wide layers."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
M32 = 0xFFFFFFFF
PAD = 64        # every tensor starts at a multiple of so many elements in the flat buffers (a 256-byte boundary in f32)
BLOCK = 32      # elements of the 8-bit states that share an exponent


def listed():
    return [
        # one lock-step move of every slot: the search's visit counts as a policy, tempered; latency
        {"name": "logp_move", "op": "logp", "rows": 4096, "actions": 2, "dtype": "f32", "logits": "visits", "mask": "none",
         "temperature": 0.5, "top": 2},
        # the recorded games of 4096 slots x 500 moves, the moves behind a game's end empty
        {"name": "logp_history", "op": "logp", "rows": 2048000, "actions": 4, "dtype": "f32", "logits": "visits",
         "mask": "none", "temperature": 1.0, "top": 1},
        # one observation answered: 17 bins in each of 4 dimensions, the 20 best alternatives
        {"name": "logp_answer", "op": "logp", "rows": 1, "actions": 83521, "dtype": "f16", "logits": "head", "mask": "shared",
         "temperature": 1.0, "top": 20},
        # an unrolled training batch over 10 bins in each of 5 dimensions
        {"name": "logp_bins", "op": "logp", "rows": 640, "actions": 100000, "dtype": "bf16", "logits": "head", "mask": "none",
         "temperature": 1.0, "top": 5},
        # loss and gradient of an unrolled training batch at the widest discrete head of the built-in models
        {"name": "grad_unroll", "op": "grad", "rows": 640, "actions": 64, "dtype": "f32", "logits": "head", "mask": "rows",
         "temperature": 1.0, "way": "given"},
        # the same through autograd, over 9 bins in each of 5 dimensions
        {"name": "grad_autograd", "op": "grad", "rows": 1280, "actions": 59049, "dtype": "f16", "logits": "head",
         "mask": "none", "temperature": 0.7, "way": "autograd"},
        # every slot's move as one training batch over 17 ** 4 actions, some of them illegal everywhere
        {"name": "grad_slots", "op": "grad", "rows": 4096, "actions": 83521, "dtype": "bf16", "logits": "head",
         "mask": "shared", "temperature": 1.0, "way": "given"},
        # the CartPole MLP's own tensors, clipped
        {"name": "adamw_mlp", "op": "adamw", "list": "mlp", "count": 16, "size": 12734, "param": "f32", "grad": "f32",
         "bits": 32, "master": False, "clip": 1.0},
        # wide layers in bf16 over fp32 master weights, clipped
        {"name": "adamw_master", "op": "adamw", "list": "layers", "count": 12, "size": 100000000, "param": "bf16",
         "grad": "bf16", "bits": 32, "master": True, "clip": 1.0},
        # f32 weights with 8-bit states, ragged sizes
        {"name": "adamw_bytes", "op": "adamw", "list": "ragged", "count": 75, "size": 64000000, "param": "f32", "grad": "f32",
         "bits": 8, "master": False, "clip": 0.0},
        # the norm of a vision model's many small tensors
        {"name": "norm_ragged", "op": "norm", "list": "ragged", "count": 150, "size": 1500000, "grad": "f32"},
        # the norm of wide layers' gradients
        {"name": "norm_layers", "op": "norm", "list": "layers", "count": 12, "size": 300000000, "grad": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logp", "logp", "grad", "grad", "adamw", "adamw", "norm"])
    if op in ("logp", "grad"):
        actions = _log_uniform(rng, 2, 200000)
        rows = _log_uniform(rng, 1, max(1, min(2000000, 150000000 // actions)))
        case = {"op": op, "rows": rows, "actions": actions, "dtype": rng.choice(sorted(DTYPES)),
                "logits": rng.choice(["head", "visits"]) if actions <= 64 else "head",
                "mask": rng.choice(["none", "shared", "rows"]), "temperature": rng.choice([1.0, round(rng.uniform(0.25, 2), 3)])}
        return {**case, "top": min(actions, rng.choice([0, 1, 5, 20, 32]))} if op == "logp" else \
            {**case, "way": rng.choice(["given", "autograd"])}
    case = {"op": op, "list": rng.choice(["layers", "ragged"]), "count": _log_uniform(rng, 1, 200),
            "size": _log_uniform(rng, 10000, 90000000), "grad": rng.choice(sorted(DTYPES))}
    if op == "norm":
        return case
    param = rng.choice(sorted(DTYPES))
    return {**case, "param": param, "grad": rng.choice([param, "f32"]), "bits": rng.choice([32, 8]),
            "master": param != "f32" and rng.choice([True, False]), "clip": rng.choice([0.0, 1.0])}


def _sizes(case):
    """Element counts of the tensors of a parameter list."""
    n, total = case["count"], case["size"]
    if case["list"] == "mlp":       # observation 4, actions 2, state 31, hidden 64, in the framework's order
        return [256, 64, 1984, 31, 2112, 64, 1984, 31, 1984, 31, 1984, 64, 128, 2, 1984, 31]
    if case["list"] == "layers":    # equal matrices, each with its bias
        side = max(1, math.isqrt(max(1, total // max(1, n // 2))))
        return [side * side if i % 2 == 0 else side for i in range(n)]
    return [max(1, int(total * 2 * (i + 1) / (n * (n + 1))) | 1) for i in range(n)]     # a ramp of odd sizes


def _layout(case):
    """(sizes, where each starts in a flat buffer, the buffer's length)."""
    sizes, at, end = _sizes(case), [], 0
    for s in sizes:
        at.append(end)
        end += -(-s // PAD) * PAD
    return sizes, at, end


def _views(flat, sizes, at):
    return [flat[a:a + s] for s, a in zip(sizes, at)]


def _policy_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, n = case["rows"], case["actions"]
    made = dict(generator=g, device="cuda")
    if case["logits"] == "visits":      # log of the children's visit counts; a tenth of the rows lie behind a game's end
        visits = torch.rand(rows, n, **made).pow_(3).mul_(50.0).floor_()
        visits[:, 0] += 1.0
        live = torch.rand(rows, 1, **made) >= 0.1
        logits = torch.log(visits * live)
        action = torch.where(live[:, 0], torch.randint(0, n, (rows,), **made), -1)
    else:                               # a trained head: a few actions stand out
        logits = torch.randn(rows, n, **made).mul_(2.0)
        action = torch.randint(0, n, (rows,), **made)
        logits.scatter_add_(1, action[:, None], torch.rand(rows, 1, **made) * 12.0)
    mask = None
    if case["mask"] == "shared":
        mask = torch.rand(n, **made) < 0.8
        mask[0] = True
    elif case["mask"] == "rows":
        mask = torch.rand(rows, n, **made) < 0.8
        mask[:, 0] = True
    s = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "action": action, "mask": mask}
    if case["op"] == "grad":            # advantages over the batch, and an entropy bonus
        s["grad_log_prob"] = torch.randn(rows, **made) / rows
        s["grad_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
        if case["way"] == "autograd":
            s["logits"].requires_grad_(True)
    return s


def _optimizer_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes, at, end = _layout(case)
    made = dict(generator=g, device="cuda")
    real = torch.zeros(end, dtype=torch.bool, device="cuda")
    for v in _views(real, sizes, at):
        v.fill_(True)
    width = torch.zeros(end, device="cuda")     # gradients of one tensor are alike, those of two differ by decades
    for v, e in zip(_views(width, sizes, at), torch.rand(len(sizes), generator=torch.Generator().manual_seed(seed)).tolist()):
        v.fill_(10.0 ** (-1 - 3 * e))
    grad = (torch.randn(end, **made) * width).to(DTYPES[case["grad"]])
    s = {"case": case, "grad": grad, "grads": _views(grad, sizes, at)}
    if case["op"] == "norm":
        return s
    weight = torch.randn(end, **made) * 0.05 * real
    first = torch.randn(end, **made) * 0.3 * width
    root = (torch.rand(end, **made) + 0.5) * width
    s |= {"param": weight.to(DTYPES[case["param"]]), "master": weight.clone() if case["master"] else None, "step": 99,
          "lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "seed": 20 + seed % 1000}
    s["params"] = _views(s["param"], sizes, at)
    if case["bits"] == 32:
        s |= {"exp_avg": first, "exp_avg_sq": root.square()}
    else:
        s["exp_avg"], s["exp_avg_exponent"] = _to_bytes(first, torch.full_like(first, 0.5))
        s["exp_avg_root"], s["exp_avg_root_exponent"] = _to_bytes(root, torch.full_like(root, 0.5))
    return s


STATES = ("exp_avg", "exp_avg_sq", "exp_avg_exponent", "exp_avg_root", "exp_avg_root_exponent", "master")


def prepare(case, seed):
    if case["op"] in ("logp", "grad"):
        return _policy_inputs(case, seed)
    s = _optimizer_inputs(case, seed)
    if own:     # what a program keeps over its steps: the list of its gradients' buffers, the optimizer (resumed at step 99)
        from muzero_amd.optim import AdamW, TensorList
        s["grads"] = TensorList(s["grads"])
        if case["op"] == "adamw":
            opt = AdamW(s["params"], lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["weight_decay"],
                        state_bits=case["bits"], master_weights=case["master"], max_grad_norm=case["clip"] or None,
                        seed=s["seed"])
            opt.load_state_dict({"step": s["step"], **{k: s[k] for k in STATES if s.get(k) is not None}})
            s["optimizer"] = opt
    return s


# ---------------------------------------------------------------------------------------------------- plain forms

def _plain_policy(s):
    """The forward values, and what the gradient needs of them."""
    case = s["case"]
    raw = s["logits"].detach().float()
    if s["mask"] is not None:
        raw = torch.where(s["mask"], raw, -math.inf)
    z = raw * (1.0 / case["temperature"])
    top = z.max(1).values
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z - top[:, None])
    total = e.sum(1)
    weighted = torch.where(e > 0, e * (z - top[:, None]), e).sum(1)
    empty = total == 0
    log_total = torch.log(total)
    log_z = top + log_total
    entropy = torch.where(empty, 0.0, log_total - weighted / total)
    a = s["action"]
    at = torch.gather(z, 1, a.clamp(min=0)[:, None])[:, 0]
    log_prob = torch.where(a < 0, 0.0, torch.where(at == -math.inf, at, (at - top) - log_total))
    return raw, z, e, total, log_z, entropy, log_prob


def _plain_top(raw, z, log_z, top):
    """Keys that order by value, then by the lower index."""
    bits = (raw + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (bits << 32) + (M32 - torch.arange(raw.shape[1], device=raw.device))
    key = key.topk(top, dim=1).values
    at = M32 - (key & M32)
    z = torch.gather(z, 1, at)
    none = z == -math.inf
    return torch.where(none, z, z - log_z[:, None]), torch.where(none, -1, at).to(torch.int32)


def _plain_grad(s, z, e, total, log_z, entropy):
    g_a = torch.where(s["action"] < 0, 0.0, s["grad_log_prob"])
    p = torch.where(total[:, None] > 0, e / total[:, None], 0.0)
    log_p = torch.where(p > 0, z - log_z[:, None], 0.0)
    d = -p * (g_a[:, None] + s["grad_entropy"][:, None] * (log_p + entropy[:, None]))
    a = s["action"].clamp(min=0)[:, None]
    here = torch.gather(z, 1, a) > -math.inf
    d.scatter_add_(1, a, g_a[:, None] * here)
    return (d * (1.0 / s["case"]["temperature"])).to(s["logits"].dtype)


def _mix(x):
    """A bijection of 32-bit words: two rounds of shift, exclusive or and an odd multiplier."""
    x = x ^ (x >> 16)
    x = (x * 0xBB67AE85) & M32
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & M32
    return x ^ (x >> 16)


def _dither(seed, step, n, device):
    """32 bits for every element of the flat state, as two numbers of 16 bits in [0, 1)."""
    key = _mix((seed & M32) ^ _mix((step * 0x9E3779B9 + (seed >> 32)) & M32))
    r = _mix((torch.arange(n, device=device) * 0x9E3779B1 + key) & M32)
    return (r >> 16).float() * 2.0 ** -16, (r & 0xFFFF).float() * 2.0 ** -16


def _to_bytes(x, r):
    """Block-scaled e4m3: per 32 elements the smallest power of two that brings the largest to 448 at most; each value rounded to the
    grid point below |x| / scale + r steps, r in [0, 1)."""
    x, r = x.view(-1, BLOCK), r.view(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True)
    f, e = torch.frexp(most)
    e = torch.where(most > 0, torch.where(f > 0.875, e - 8, e - 9), -127).clamp(min=-127)
    y = torch.ldexp(torch.ldexp(x.abs(), -(e // 2)), -(e - e // 2))
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)
    y = torch.copysign(torch.floor(y / step + r) * step, x)
    return y.reshape(-1).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(-1).view(torch.float8_e8m0fnu)


def _from_bytes(code, exponent):
    return (code.float().view(-1, BLOCK) * exponent.float().view(-1, 1)).view(-1)


def _plain_norm(s):
    return s["grad"].float().square().sum(dtype=torch.float64).sqrt().float()


def _plain_adamw(s):
    case, (b1, b2) = s["case"], s["betas"]
    s["step"] += 1
    norm = _plain_norm(s) if case["clip"] else None
    g = s["grad"].float()
    if case["clip"]:
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1.0)
    if case["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = _from_bytes(s["exp_avg"], s["exp_avg_exponent"])
        v = _from_bytes(s["exp_avg_root"], s["exp_avg_root_exponent"]).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    step_size, root_2 = s["lr"] / (1 - b1 ** s["step"]), 1 / math.sqrt(1 - b2 ** s["step"])
    w = s["param"].float() if s["master"] is None else s["master"]
    root = v.sqrt()
    w = w * (1 - s["lr"] * s["weight_decay"]) - step_size * (m / (root * root_2 + s["eps"]))
    s["param"].copy_(w)
    if s["master"] is not None:
        s["master"].copy_(w)
    if case["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return norm
    r1, r2 = _dither(s["seed"], s["step"], m.numel(), m.device)
    for name, x, r in (("exp_avg", m, r1), ("exp_avg_root", root, r2)):
        code, exponent = _to_bytes(x, r)
        if name == "exp_avg_root":      # a root that is not zero keeps the smallest code
            code = torch.where((code.float() == 0) & (x > 0), 2.0 ** -9, code.float()).to(code.dtype)
        s[name].copy_(code)
        s[name + "_exponent"].copy_(exponent)
    return norm


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        return [_plain_norm(s)]
    if case["op"] == "adamw":
        norm = _plain_adamw(s)
        return {"param": s["param"], "norm": norm, **{k: s[k] for k in STATES if s.get(k) is not None}}
    raw, z, e, total, log_z, entropy, log_prob = _plain_policy(s)
    if case["op"] == "grad":
        return [log_prob, entropy, log_z, _plain_grad(s, z, e, total, log_z, entropy)]
    top = _plain_top(raw, z, log_z, case["top"]) if case["top"] else ()
    return [log_prob, entropy, log_z, *top]


def run(s):
    if not own:
        return _plain(s)
    case = s["case"]
    if case["op"] == "norm":
        from muzero_amd.optim import grad_norm
        return [grad_norm(s["grads"])]
    if case["op"] == "adamw":
        opt = s["optimizer"]
        opt.step(s["grads"])
        return {"param": s["param"], "norm": opt.grad_norm if case["clip"] else None, **opt.state_tensors()}
    from muzero_amd.policy import policy_log_probs, policy_log_probs_grad
    given = dict(mask=s["mask"], temperature=case["temperature"])
    if case["op"] == "grad":
        if case["way"] == "given":
            out, grad = policy_log_probs_grad(s["logits"], s["action"], s["grad_log_prob"], s["grad_entropy"], **given)
        else:
            out = policy_log_probs(s["logits"], s["action"], **given)
            grad, = torch.autograd.grad((out.log_prob, out.entropy), s["logits"], (s["grad_log_prob"], s["grad_entropy"]))
        return [out.log_prob.detach(), out.entropy.detach(), out.log_z.detach(), grad]
    out = policy_log_probs(s["logits"], s["action"], top=case["top"], **given)
    return [out.log_prob, out.entropy, out.log_z] + ([out.top_log_prob, out.top_action] if case["top"] else [])


def work(case):
    if case["op"] in ("logp", "grad"):
        rows, n = case["rows"], case["actions"]
        one = rows * n * BYTES[case["dtype"]]
        mask = {"none": 0, "shared": n, "rows": rows * n}[case["mask"]]
        if case["op"] == "grad":
            return {"bytes": 2 * one + mask + rows * 28, "flops": 12 * rows * n}
        return {"bytes": one + mask + rows * (20 + 8 * case["top"]), "flops": 6 * rows * n}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": n * BYTES[case["grad"]] + 4, "flops": 2 * n}
    # gradient read; weight read and written (or only written, beside the master weight's read and write); two states
    weight = BYTES[case["param"]] + 8 if case["master"] else 2 * BYTES[case["param"]]
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    return {"bytes": n * (BYTES[case["grad"]] + weight + state), "flops": 20 * n}


# ------------------------------------------------------------------------------- the definitions, in 64 bits

def _exact_policy(case, s):
    l = s["logits"].detach().double()
    n = l.shape[1]
    legal = torch.ones_like(l, dtype=torch.bool) if s["mask"] is None else s["mask"].expand_as(l)
    l = l.masked_fill(~legal, -math.inf)
    z = l / case["temperature"]
    log_z = torch.logsumexp(z, 1)
    filled = log_z > -math.inf
    log_p = (z - torch.where(filled, log_z, 0.0)[:, None])
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    a = s["action"]
    rows = torch.arange(l.shape[0], device=l.device)
    log_prob = torch.where(a >= 0, log_p[rows, a.clamp(min=0)], 0.0)
    out = [log_prob, entropy, log_z]
    if case["op"] == "grad":
        g_a, g_h = s["grad_log_prob"].double() * (a >= 0), s["grad_entropy"].double()
        chosen = torch.zeros_like(p)
        chosen[rows, a.clamp(min=0)] = g_a
        chosen = chosen.masked_fill(l == -math.inf, 0.0)
        inside = torch.where(p > 0, p * (g_h[:, None] * (torch.where(p > 0, log_p, 0.0) + entropy[:, None]) + g_a[:, None]), 0.0)
        return out + [(chosen - inside) / case["temperature"]]
    if case["top"]:
        values, index = torch.sort(l, dim=1, descending=True, stable=True)
        values, index = values[:, :case["top"]] / case["temperature"], index[:, :case["top"]]
        none = values == -math.inf
        out += [torch.where(none, values, values - torch.where(filled, log_z, 0.0)[:, None]),
                index.masked_fill(none, -1).to(torch.int32)]
    return out


def _exact_bytes(x, r):
    """The grid of e4m3 below 448: steps of 2 ** -9 up to 2 ** -6, from there 8 steps to the octave."""
    b = x.view(-1, BLOCK)
    most = b.abs().amax(1)
    exponent = torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / 448))
    exponent = torch.where(most * torch.exp2(-exponent) > 448, exponent + 1, exponent)
    exponent = torch.where(most * torch.exp2(1 - exponent) <= 448, exponent - 1, exponent)
    exponent = torch.where(most > 0, exponent, -127.0).clamp(min=-127)
    y = b.abs() * torch.exp2(-exponent)[:, None]
    octave = torch.frexp(y).exponent.clamp(min=-5) - 1
    grid = torch.exp2((octave - 3).double())
    y = torch.floor(y / grid + r.view(-1, BLOCK).double()) * grid
    return torch.where(b < 0, -y, y).view(-1), torch.exp2(exponent)


def _exact_optimizer(case, s):
    g = s["grad"].double()
    norm = torch.sqrt((g * g).sum())
    if case["op"] == "norm":
        return [norm]
    t, (b1, b2) = s["step"] + 1, s["betas"]
    if case["clip"]:
        g = g * min(1.0, case["clip"] / (norm.item() + 1e-6))
    if case["bits"] == 32:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        m = (s["exp_avg"].double().view(-1, BLOCK) * s["exp_avg_exponent"].double()[:, None]).view(-1)
        v = (s["exp_avg_root"].double().view(-1, BLOCK) * s["exp_avg_root_exponent"].double()[:, None]).view(-1) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    w = (s["param"] if s["master"] is None else s["master"]).double()
    w = w - s["lr"] * (s["weight_decay"] * w + (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + s["eps"]))
    out = {"param": w, "norm": norm if case["clip"] else None}
    if s["master"] is not None:
        out["master"] = w
    if case["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    r1, r2 = _dither(s["seed"], t, m.numel(), m.device)
    out["exp_avg"], out["exp_avg_exponent"] = _exact_bytes(m, r1)
    out["exp_avg_root"], out["exp_avg_root_exponent"] = _exact_bytes(v.sqrt(), r2)
    out["exp_avg_root"] = torch.where((out["exp_avg_root"] == 0) & (v > 0), 2.0 ** -9, out["exp_avg_root"])
    return out


def exact(case, seed):
    if case["op"] in ("logp", "grad"):
        return _exact_policy(case, _policy_inputs(case, seed))
    return _exact_optimizer(case, _optimizer_inputs(case, seed))
