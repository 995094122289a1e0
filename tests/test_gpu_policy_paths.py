"""Policy log-probabilities and AdamW where the framework itself calls them - Trainer(optimizer="adamw"), Muzero.policy_statistics,
Arena.policy_statistics - and the operators together, as a training step of a wide policy head runs them.

Tolerances, u = 2^-24.  AdamW over s <= 3 steps: |m_hat| / sqrt(v_hat) <= 1.02 (Cauchy's inequality, both averages over the same gradients
with nearly equal weights), so a step is at most 1.02 lr; its rounding is 9 u of that, 4 u a step from m, 5 u a step from v and 8 u
from the clipping factor: under 60 u lr a step; w (1 - lr wd) - step adds 2 u |w|."""
import numpy as np
import pytest
import torch

from conftest import load_golden

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def adamw64(w, m, v, g, t, lr, wd, max_norm, b1=0.9, b2=0.999, eps=1e-8):
    norm = np.sqrt((g * g).sum())
    if max_norm:
        g = g * min(1.0, max_norm / (norm + 1e-6))
    m[:] = b1 * m + (1 - b1) * g
    v[:] = b2 * v + (1 - b2) * g * g
    return w * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)


def trainer(fixture, precision=None, **kw):
    from muzero_amd.engine import SearchEngine
    from muzero_amd.train import Trainer
    fx = load_golden(fixture + ".npz")
    dims = tuple(int(x) for x in fx["dims"])
    dims = dims + (2,) if "vis" in fixture else dims + (0, precision) if precision else dims
    eng = SearchEngine(dims, max_games=4, max_simulations=0)
    eng.set_weights(fx["blob0"])
    return fx, eng, Trainer(eng, int(fx["K"]), int(fx["B"]), "adamw", 0.01, **kw)


def statistics(fx, n):
    """which blob elements are running statistics of BatchNorm"""
    if fx["dims"].size != 5 or int(fx["dims"][0]) == 4:
        return np.zeros(n, bool)
    from test_vision_train_oracle import vo
    _, A, Sd, H, L = [int(x) for x in fx["dims"]]
    return np.concatenate([np.full(int(np.prod(s)), name.endswith(("_var", "_mean"))) for name, s in vo.blob_layout(A, Sd, H, L)])


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("fixture", ["train_tag123_K5_B128", "train_lstmB_K3_B32", "train_visB_K2_B4"])
def test_trainer_steps(fixture, max_norm):
    fx, eng, tr = trainer(fixture, weight_decay=0.1, max_grad_norm=max_norm)
    w = tr.weights().astype(np.float64)
    stat = statistics(fx, w.size)
    assert stat.any() == ("vis" in fixture)
    m, v = np.zeros((~stat).sum()), np.zeros((~stat).sum())
    g = torch.Generator().manual_seed(5)
    for t in range(1, 4):
        grad = torch.randn(w.size, generator=g) * 0.01
        grad[torch.from_numpy(stat)] *= 0.1
        tr.grad.copy_(grad)
        tr.apply()
        grad = grad.double().numpy()
        w[stat] += grad[stat]
        w[~stat] = adamw64(w[~stat], m, v, grad[~stat], t, 0.01, 0.1, max_norm)
        got = tr.weights()
        assert np.all(np.abs(got - w) <= t * (60 * U * 0.01 + 2 * U * np.abs(w)) + U * np.abs(w))
        if max_norm and t < 3:            # a step that is not finite leaves everything, the step count too
            tr.grad[int(np.flatnonzero(~stat)[-1])] = float("nan") if t == 1 else float("inf")
            tr.apply()
            assert np.array_equal(tr.weights(), got)
    eng.close()


@pytest.mark.parametrize("fixture, precision", [("train_tag123_K5_B128", None), ("train_tag123_K5_B128", 1), ("train_tag123_K5_B128", 2),
                                                ("train_lstmB_K3_B32", None), ("train_visB_K2_B4", None)])
def test_inference_follows_the_trainer(fixture, precision):
    from muzero_amd.engine import SearchEngine
    fx, eng, tr = trainer(fixture, precision, max_grad_norm=1.0)
    tr.grad.copy_(torch.randn(tr.grad.numel(), generator=torch.Generator().manual_seed(1)).abs() * 0.01)
    tr.apply()
    blob = tr.weights()
    assert np.count_nonzero(blob != fx["blob0"]) > 0.9 * blob.size
    other = SearchEngine(eng.dims, max_games=4, max_simulations=0)
    other.set_weights(blob)
    if "vis" in fixture:
        from test_vision_train_oracle import step_inputs
        obs = step_inputs(fx, 0)["obs"][:3]
    else:
        obs = fx["s0_obs"][:3]
    for x, y in zip(eng.initial_inference(obs), other.initial_inference(obs)):
        assert torch.equal(x, y)
    eng.close(), other.close()


def test_trainer_follows_the_momentum_schedule():
    """onecyclelr moves beta1 with the rate, of AdamW as of Adam."""
    from muzero_amd.train import scheduled_lr, scheduled_momentum
    fx, eng, tr = trainer("train_tag123_K5_B128", weight_decay=0.05, lr_scheduler="onecyclelr", num_of_epoch=20)
    w = tr.weights().astype(np.float64)
    m, v, beta = np.zeros_like(w), np.zeros_like(w), []
    for t in range(1, 4):
        grad = torch.randn(w.size, generator=torch.Generator().manual_seed(t)) * 0.01
        tr.grad.copy_(grad)
        lr, b1 = scheduled_lr("onecyclelr", 0.01, 20, t - 1), scheduled_momentum("onecyclelr", 20, t - 1)
        beta.append(b1)
        tr.apply()
        w = adamw64(w, m, v, grad.double().numpy(), t, lr, 0.05, None, b1=b1)
        # beta1 below 0.95 and three steps: bias corrections as before, averages over the same three gradients
        assert np.all(np.abs(tr.weights() - w) <= t * (60 * U * 0.01 + 2 * U * np.abs(w)) + U * np.abs(w))
    assert len(set(beta)) > 1
    eng.close()


def test_trainer_refusals():
    from muzero_amd import _lib
    from muzero_amd.engine import SearchEngine
    from muzero_amd.train import Trainer
    fx = load_golden("train_tag123_K5_B128.npz")
    eng = SearchEngine(tuple(int(x) for x in fx["dims"]), max_games=1, max_simulations=0)
    eng.set_weights(fx["blob0"])
    for kw in (dict(optimizer="adamw", weight_decay=-0.1), dict(optimizer="adamw", weight_decay=float("nan")),
               dict(optimizer="adamw", max_grad_norm=0.0), dict(optimizer="adam", max_grad_norm=1.0), dict(optimizer="lion")):
        with pytest.raises(ValueError):
            Trainer(eng, 5, 8, **kw)
    with pytest.raises(_lib.MzsError):                       # no trainer yet
        _lib.check(eng.lib.mzs_train_set_adamw(eng.h, 0.999, 1e-8, 0.0, 0.0), "set_adamw")
    tr = Trainer(eng, 5, 8, "adam")
    tr.opt = "adamw"                                         # its states were never made
    with pytest.raises(_lib.MzsError):
        tr.apply()
    with pytest.raises(_lib.MzsError):
        _lib.check(eng.lib.mzs_train_set_adamw(eng.h, 1.0, 1e-8, 0.0, 0.0), "set_adamw")
    eng.close()


def test_muzero_trains_with_adamw_and_keeps_its_options(tmp_path):
    from muzero_amd.model import Muzero
    fx = load_golden("train_tag123_K5_B128.npz")
    mz = Muzero(model_structure="mlp_model", observation_space_dimensions=4, action_space_dimensions=2, state_space_dimensions=31,
                hidden_layer_dimensions=64, number_of_hidden_layer=0, k_hypothetical_steps=5, learning_rate=0.01, optimizer="adamw")
    mz.optimizer_options = {"weight_decay": 0.05, "max_grad_norm": 1.0}
    mz.set_weights(fx["blob0"])
    K, B, A = fx["s0_actions"].shape
    batch = []
    for b in range(B):
        acts = [fx["s0_actions"][k, b] for k in range(K)]
        tg = [[float(fx["s0_target_value"][k, b]), float(fx["s0_target_reward"][k, b]), fx["s0_target_policy"][k, b]] for k in range(K)]
        batch.append((torch.tensor(fx["s0_obs"][b:b + 1]), acts, tg))
    pos = np.stack([np.arange(B), np.arange(B)], axis=1)
    before = mz.weights_blob().astype(np.float64)
    mz.train((batch, fx["s0_is_ratio"], pos))
    grad = mz._trainer.grad.cpu().numpy().astype(np.float64)
    w = adamw64(before, np.zeros_like(before), np.zeros_like(before), grad, 1, 0.01, 0.05, 1.0)
    assert np.all(np.abs(mz.weights_blob() - w) <= 60 * U * 0.01 + 3 * U * np.abs(w))
    mz.save_model(str(tmp_path), tag=7, model_update_condition=True)
    other = Muzero(load=True)
    other.load_model(str(tmp_path), tag=7)
    assert other.opt == "adamw" and other.optimizer_options == mz.optimizer_options


def test_model_statistics():
    from muzero_amd.model import Muzero
    fx = load_golden("train_tag123_K5_B128.npz")
    mz = Muzero(model_structure="mlp_model", observation_space_dimensions=4, action_space_dimensions=2, state_space_dimensions=31,
                hidden_layer_dimensions=64, number_of_hidden_layer=0)
    mz.set_weights(fx["blob0"])
    obs = fx["s0_obs"][:17]
    p = mz._inference_engine().initial_inference(obs)[1].double().cpu().numpy()
    actions = np.arange(17) % 2
    for temperature in (1.0, 0.5):
        q = p ** (1 / temperature)
        z = q.sum(1)
        out = mz.policy_statistics(obs, actions, temperature=temperature, top=2)
        # the logits are rounded logarithms: u |log p| each, 8 u for the operator's exponentials and logarithm
        tol = (8 + 2 * np.abs(np.log(p)).max() / temperature) * U * 4
        assert np.allclose(out.log_prob.cpu(), np.log(q / z[:, None])[np.arange(17), actions], rtol=0, atol=tol)
        assert np.allclose(out.log_z.cpu(), np.log(z), rtol=0, atol=tol)
        assert np.allclose(out.entropy.cpu(), -(q / z[:, None] * np.log(q / z[:, None])).sum(1), rtol=0, atol=tol)
        assert np.array_equal(out.top_action.cpu(), np.argsort(-p, axis=1, kind="stable"))
    assert float(mz.policy_statistics(obs).log_prob.abs().max()) == 0.0


def test_arena_statistics():
    from muzero_amd.selfplay import Arena
    from test_gpu_selfplay import fake_results, make_engine
    G, T = 24, 12
    eng, _, _ = make_engine(G, 0)
    ar = Arena(eng, G, 2 * G, T)
    ar.begin(G, np.arange(G, dtype=np.int64) * 31 + 5, episode=0)
    rs = np.random.RandomState(3)
    for _ in range(T):
        res = fake_results(rs, G, 2, eng.device)[1]
        ar.step(1.0, res, num_simulations=50)
        if int(ar.alive_count.item()) == 0:
            break
    length, action = ar.arrays["length"].cpu().numpy(), ar.arrays["action"].cpu().numpy()
    pi = ar.arrays["policy"].cpu().numpy().astype(np.float64)
    row0, n = G + 3, G - 5
    out = ar.policy_statistics(row0, n, temperature=0.5, top=1)
    assert out.log_prob.shape == (n, T) and out.top_action.shape == (n, T, 1)
    assert length[row0:row0 + n].min() >= 1 and length[row0:row0 + n].max() <= T
    for r in range(n):
        for t in range(T):
            lp, lz, h = (float(x[r, t]) for x in (out.log_prob, out.log_z, out.entropy))
            if t >= length[row0 + r]:
                assert lp == 0.0 and lz == -np.inf and h == 0.0 and int(out.top_action[r, t, 0]) == -1
                continue
            q = pi[row0 + r, t] ** 2
            q /= q.sum()
            logs = np.abs(np.log(pi[row0 + r, t][pi[row0 + r, t] > 0])).max()
            tol = (8 + 4 * logs) * U * 4
            assert lp == np.log(q[action[row0 + r, t]]) or abs(lp - np.log(q[action[row0 + r, t]])) <= tol
            assert abs(h + sum(x * np.log(x) for x in q if x > 0)) <= tol
            assert int(out.top_action[r, t, 0]) == int(np.argmax(q))
    for bad in ((-1, 2), (0, 0), (G, G + 1)):
        with pytest.raises(ValueError):
            ar.policy_statistics(*bad)
    ar.close(), eng.close()


def test_operators_together():
    """Three training steps of a policy head over 257 actions with masks, as a program runs them: logits, log-probabilities and entropy,
    their gradient, the clipped step - against the same in 64 bits from the same weights.

    Logits: 48 products and sums, 48 u of sum |x w|.  The gradient of a logit, at most 2 (|g| + |h| (10 + |H|)) / rows here, is off by that
    error of the exponents times itself and 32 u; a weight's gradient sums 64 rows of them: bounded by (64 + 32 + 2 * 48 * max sum |x w|) u
    times sum |x| bound."""
    from muzero_amd.optim import AdamW
    from muzero_amd.policy import policy_log_probs
    rows, width, n = 64, 48, 257
    g = torch.Generator().manual_seed(11)
    x = torch.randn(rows, width, generator=g).cuda()
    w = (torch.randn(width, n, generator=g) * 0.2).cuda().requires_grad_()
    b = (torch.randn(n, generator=g) * 0.2).cuda().requires_grad_()
    mask = (torch.rand(rows, n, generator=g) < 0.8)
    mask[5] = False
    actions = torch.where(mask.any(1), mask.int().argmax(1), -1)
    opt = AdamW([w, b], lr=0.01, weight_decay=0.1, max_grad_norm=0.05)
    state = [[np.zeros(p.shape), np.zeros(p.shape)] for p in (w, b)]
    for t in range(1, 4):
        w64, b64 = (p.detach().double().cpu().requires_grad_() for p in (w, b))
        x64 = x.double().cpu()
        logits = (x64 @ w64 + b64) / 0.7
        some = mask.any(1)
        lp = torch.log_softmax(logits.masked_fill(~mask, -torch.inf)[some], 1)
        h = -(lp.exp() * lp.masked_fill(~mask[some], 0.0)).sum(1)
        (-(lp.gather(1, actions[some][:, None]).sum() + 0.01 * h.sum()) / rows).backward()
        out = policy_log_probs(x @ w + b, actions.cuda(), mask=mask.cuda(), temperature=0.7)
        loss = -(out.log_prob.sum() + 0.01 * out.entropy.sum()) / rows
        opt.zero_grad()
        loss.backward()
        products = float((x64.abs() @ w64.abs() + b64.abs()).max().detach()) / 0.7
        bound = 2 * (1 + 0.01 * 20) / 0.7 / rows
        for p, q, load in ((w, w64, float(x64.abs().sum(0).max())), (b, b64, float(rows))):
            assert float((p.grad.double().cpu() - q.grad).abs().max()) <= (96 + 2 * 48 * products) * U * load * bound
        before = [p.detach().double().cpu().numpy() for p in (w, b)]
        grads = [p.grad.double().cpu().numpy() for p in (w, b)]
        norm = np.sqrt(sum((q * q).sum() for q in grads))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 8 * U * norm and norm > 0.05
        for p, old, q, (m, v) in zip((w, b), before, grads, state):
            want = adamw64(old, m, v, q * min(1.0, 0.05 / (norm + 1e-6)), t, 0.01, 0.1, 0.0)
            assert np.all(np.abs(p.detach().cpu().numpy() - want) <= 60 * U * 0.01 * t + 3 * U * np.abs(want))


@pytest.mark.parametrize("name, precision", [("tag123", 0), ("tag137", 0), ("lstmA", 0), ("visA", 0), ("tag123", 1)])
def test_logits_of_the_policy_head(name, precision):
    """Their softmax is initial_inference's policy: 3 roundings of the exponent, 8 of exponential, sum and quotient on each side."""
    from conftest import fixture_weights
    from muzero_amd.engine import SearchEngine
    d, blob = fixture_weights(name)
    obs = np.random.RandomState(3).uniform(-1, 1, size=(5, 3, 98, 98) if name == "visA" else (37, d.obs_dim)).astype(np.float32)
    eng = SearchEngine((d.obs_dim, d.n_actions, d.state_dim, d.hidden_dim, d.n_mid_layers, d.model_kind, precision),
                       max_games=len(obs), max_simulations=0)
    eng.set_weights(blob)
    logits, p = eng.initial_logits(obs).double(), eng.initial_inference(obs)[1].double()
    want = torch.log_softmax(logits, 1)
    assert float((want.exp() - p).abs().max()) <= (16 + 4 * float(logits.abs().max())) * U and float(logits.std()) > 0
    eng.close()


def test_model_statistics_of_a_head_that_is_sure():
    """Policies with probabilities below e^-87, where the inference's softmax ends: they have a log-probability, and count at temperatures
    above 1.  The policy head's weights 2^10 times as large give logits of exactly 2^10 times; u of the largest logit for each of their three
    roundings behind it."""
    from muzero_amd.model import Muzero
    fx = load_golden("train_tag123_K5_B128.npz")
    mz = Muzero(model_structure="mlp_model", observation_space_dimensions=4, action_space_dimensions=2, state_space_dimensions=31,
                hidden_layer_dimensions=64, number_of_hidden_layer=0)
    mz.set_weights(fx["blob0"])
    obs = fx["s0_obs"][:33]
    logits = mz._inference_engine().initial_logits(obs).double().cpu().numpy()
    H, A, Sd = 64, 2, 31
    blob = np.array(fx["blob0"])
    # behind the representation, dynamics and the prediction's first layer: A x H weights and A biases of the policy
    head = len(blob) - (A * H + A + Sd * H + Sd)
    blob[head:head + A * H + A] *= 1024.0
    mz.set_weights(blob)
    sure = mz._inference_engine().initial_logits(obs).double().cpu().numpy()
    assert np.array_equal(sure, 1024.0 * logits)
    p = mz._inference_engine().initial_inference(obs)[1].cpu().numpy()
    actions = np.argmin(sure, axis=1)
    logs = sure - np.logaddexp.reduce(sure, axis=1)[:, None]
    assert (np.log(p[np.arange(33), actions]) > logs[np.arange(33), actions] + 100.0).any()
    for temperature in (1.0, 10.0, 300.0):
        z = logs / temperature
        lz = np.logaddexp.reduce(z, axis=1)
        q = z - lz[:, None]
        out = mz.policy_statistics(obs, actions, temperature=temperature, top=2)
        tol = (32 + 8 * np.abs(sure).max() / temperature) * U
        assert np.abs(out.log_prob.cpu().numpy() - q[np.arange(33), actions]).max() <= tol
        assert np.abs(out.log_z.cpu().numpy() - lz).max() <= tol
        assert np.abs(out.entropy.cpu().numpy() + (np.exp(q) * q).sum(1)).max() <= tol
        assert np.array_equal(out.top_action.cpu().numpy(), np.argsort(-sure, axis=1, kind="stable"))
