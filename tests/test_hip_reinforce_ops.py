"""The operators together, as a REINFORCE step uses them: rules on the scores with the links of a first draw, paths drawn from the
result, the gradient back through the rules, and a clipped AdamW step."""
import os
import shutil

import numpy as np
import pytest
import torch

from conftest import GOLDEN
from oracle import adamw_oracle, logits_oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def graphs(B, V, C, seed=3):
    from src.common.synthetic import make_batch
    b = make_batch(B, V, C, "nsfnet" if V == 14 else "random", seed=seed)
    t = lambda k: torch.from_numpy(b[k]).to("cuda:0")
    return t("edges_capacity"), t("commodities")


def test_rules_equal_the_formula_on_drawn_paths(dev):
    from src.gcn.algorithms.path_sampler import PathSampler
    from src.gcn.algorithms.score_rules import LinkScoreRules
    B, V, C = 5, 14, 6
    cap, comm = graphs(B, V, C)
    y = torch.randn(B, V, V, C, device=dev, generator=torch.Generator(dev).manual_seed(0))
    paths, plen = PathSampler(y, cap, comm).draw()
    assert paths.shape == (B, C, 14) and not paths.requires_grad
    bias = torch.randn(V, V, device=dev)
    got = LinkScoreRules(cap, 1.5, 0.2, 0.4, bias=bias, temperature=0.7)(y, paths, plen)
    p, n = paths.cpu().numpy(), plen.cpu().numpy()
    hist = np.full((B * V, C), -1)
    for b in range(B):
        for c in range(C):
            for here, there in zip(p[b, c, :n[b, c]], p[b, c, 1:n[b, c]]):
                hist[b * V + here, c] = there
    mask = ((cap > 0) & ~torch.eye(V, dtype=torch.bool, device=dev)).cpu().numpy().reshape(B * V, V)
    want, _, _, bound = logits_oracle.process(y.cpu().double().numpy().reshape(B * V, V, C), hist, rho=1.5, alpha_p=0.2, alpha_f=0.4,
                                              bias=bias.cpu().numpy(), mask=mask, tau=0.7, masked=float(np.float32(-1e9)))
    assert (np.abs(got.cpu().double().numpy().reshape(want.shape) - want) <= 8 * U * bound).all()
    # what comes out is taken where scores are: the sampler and the beam search
    from src.gcn.algorithms.beamsearch_uelb import BeamSearchFactory
    again, _ = PathSampler(got, cap, comm).draw()
    assert again.shape == paths.shape
    bs = BeamSearchFactory.create_algorithm("unconstrained", y_pred_edges=got, beam_size=3, batch_size=B, edges_capacity=cap, commodities=comm,
                                            dtypeFloat=torch.float, dtypeLong=torch.long, mode_strict=True)
    found, _ = bs.search()
    assert len(found) == B
    for bad in (dict(paths=paths), dict(paths=paths[:2], path_len=plen[:2])):
        with pytest.raises(ValueError):
            LinkScoreRules(cap)(y, **bad)
    with pytest.raises(ValueError):
        LinkScoreRules(cap)(y[:, :, :5])


@pytest.mark.parametrize("bits", [32, 8])
def test_policy_gradient_step_through_all_operators(dev, bits):
    """Scores that are parameters: their gradient is the sampler's times the rules' slope, and the step is the formula's."""
    from src.gcn.algorithms.path_sampler import PathSampler
    from src.gcn.algorithms.score_rules import LinkScoreRules
    from src.gcn.hip.fused_adamw import FusedAdamW
    B, V, C = 4, 14, 7
    cap, comm = graphs(B, V, C)
    y = torch.nn.Parameter(torch.randn(B, V, V, C, device=dev, generator=torch.Generator(dev).manual_seed(1)))
    bias = torch.nn.Parameter(0.1 * torch.randn(V, V, device=dev, generator=torch.Generator(dev).manual_seed(2)))
    opt = FusedAdamW([y, bias], lr=1e-2, weight_decay=0.1, state_bits=bits, max_grad_norm=0.05)
    first = PathSampler(y, cap, comm).draw()
    rules = LinkScoreRules(cap, 1.3, 0.1, 0.2, bias=bias, temperature=0.8)
    used = rules(y, *first)
    sampler = PathSampler(used, cap, comm, temperature=1.2, top_p=0.9, entropy_epsilon=0.05)
    _, logp, _, _ = sampler.sample()
    advantage = torch.linspace(-1, 1, B, device=dev)
    (-logp * advantage).mean().backward()
    # the sampler's gradient on its own, then the rules' by the oracle
    leaf = used.detach().requires_grad_()
    _, logp2, _, _ = PathSampler(leaf, cap, comm, temperature=1.2, top_p=0.9, entropy_epsilon=0.05).evaluate(sampler.paths_tensor, sampler.path_len)
    (-logp2 * advantage).mean().backward()
    from src.gcn.algorithms.score_rules import hops_from
    mask = ((cap > 0) & ~torch.eye(V, dtype=torch.bool, device=dev)).cpu().numpy().reshape(B * V, V)
    _, slope, slope_b, _ = logits_oracle.process(y.detach().cpu().double().numpy().reshape(B * V, V, C),
                                                 hops_from(*first, V).cpu().numpy().reshape(B * V, C), rho=1.3, alpha_p=0.1, alpha_f=0.2,
                                                 bias=bias.detach().cpu().numpy(), mask=mask, tau=0.8)
    dx, db, size = logits_oracle.gradient(leaf.grad.cpu().double().numpy().reshape(B * V, V, C), slope, slope_b, V)
    got = y.grad.cpu().double().numpy().reshape(dx.shape)
    assert np.abs(dx).max() > 0 and (np.abs(got - dx) <= 4 * U * np.abs(dx)).all()
    assert (np.abs(bias.grad.cpu().double().numpy() - db) <= (B * C + 2) * U * size).all()
    # the update
    before = [p.detach().cpu().double().numpy().copy() for p in (y, bias)]
    grads = [p.grad.cpu().double().numpy() for p in (y, bias)]
    opt.step()
    norm = np.sqrt(sum((g ** 2).sum() for g in grads))
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    scale = min(1.0, 0.05 / (norm + 1e-6))
    assert scale < 1
    for p, old, g in zip((y, bias), before, grads):
        want, m, v = adamw_oracle.step(old, g, 0 * g, 0 * g, t=1, lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=0.1, scale=scale)
        # 4 u |p| + 20 u of the update, and 4 u more of the gradient's scale (norm and coefficient, rounded)
        step = 1e-2 * np.abs(m) / 0.1 / (np.sqrt(v / 0.001) + 1e-8)
        assert (np.abs(p.detach().cpu().double().numpy() - want) <= 4 * U * np.abs(want) + 28 * U * step + 1e-45).all()
    assert ("exp_avg_exp" in opt.state[y]) == (bits == 8)


def _strategy(dev, optimizer, **extra):
    from src.common.config.config import Settings
    from src.common.data_management.dataset_reader import DotDict
    from src.common.synthetic import make_batch
    from src.gcn.models.gcn_model import ResidualGatedGCNModel
    from src.gcn.train.trainer import make_optimizer
    from src.gcn.training.reinforcement_strategy import ReinforcementLearningStrategy
    B, V, C = 6, 14, 5
    cfg = Settings(dict(num_nodes=V, num_commodities=C, voc_edges_in=3, voc_edges_out=1, hidden_dim=32, num_layers=2, mlp_layers=2,
                        aggregation="mean", batch_size=B, beam_size=3, rl_beam_search_type="unconstrained", learning_rate=1e-3,
                        optimizer=optimizer, **extra))
    torch.manual_seed(3)
    net = ResidualGatedGCNModel(cfg, torch.float32, torch.long).to(dev).train()
    strat = ReinforcementLearningStrategy(cfg)
    data = strat.prepare_batch_data(DotDict(make_batch(B, V, C, "nsfnet", seed=9)), dev)
    return net, make_optimizer(cfg, net.parameters()), strat, data


@pytest.mark.parametrize("optimizer", ["adam", "adamw", "adamw8bit"])
def test_reinforce_steps_with_link_penalties(dev, optimizer):
    net, opt, strat, data = _strategy(dev, optimizer, rl_link_repetition_penalty=1.5, rl_link_frequency_penalty=0.3)
    before = [p.detach().clone() for p in net.parameters()]
    for step in range(3):
        loss, m = strat.compute_loss(net, data, dev)
        assert np.isfinite(loss.item()) and not m["reinforce_fallback_used"]
        assert strat.backward_step(loss, opt, 1, step)
    assert len(strat.grad_norm_history) == 3 and np.isfinite(strat.grad_norm_history).all()
    assert any(not torch.equal(a, b.detach()) for a, b in zip(before, net.parameters()))
    net.eval()
    with torch.no_grad():
        loss, m = strat.compute_loss(net, data, dev)
    assert m["reinforce_fallback_used"] and np.isfinite(loss.item())


def test_neutral_penalties_and_the_default_optimizer_change_nothing(dev):
    """The same steps with the configuration keys at their neutral values and without them: equal bits."""
    from src.gcn.hip import lib as L
    results = []
    for extra in ({}, dict(rl_link_repetition_penalty=1.0, rl_link_presence_penalty=0.0, rl_link_frequency_penalty=0.0)):
        net, opt, strat, data = _strategy(dev, "adam", **extra)
        torch.manual_seed(11)
        L.reseed()
        loss, _ = strat.compute_loss(net, data, dev)
        strat.backward_step(loss, opt, 1, 0)
        results.append([loss.detach()] + [p.detach().clone() for p in net.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_fused_clipping_in_the_strategy_equals_torch_clipping(dev):
    """backward_step with FusedAdamW (clipping inside the step) against torch's clip_grad_norm_ and the same optimizer without it."""
    from src.gcn.hip.fused_adamw import FusedAdamW
    outs = []
    for inside in (True, False):
        net, opt, strat, data = _strategy(dev, "adamw", rl_grad_clip_max_norm=0.01)
        for k, p in enumerate(net.parameters()):
            p.grad = torch.randn(p.shape, device=dev, generator=torch.Generator(dev).manual_seed(k))
        params = list(net.parameters())
        want = float(torch.sqrt(sum((p.grad.double() ** 2).sum() for p in params)))
        if inside:
            loss = sum((p * p.grad.clone()).sum() for p in params)
            for p in params:
                p.grad = None
            assert strat.backward_step(loss, opt, 1, 0)
            assert abs(strat.grad_norm_history[-1] - want) <= 2 * U * want
            assert all(p.grad is None for p in params)
        else:
            torch.nn.utils.clip_grad_norm_(params, 0.01)
            opt.step()
        outs.append([p.detach().clone() for p in params])
    for a, b in zip(*outs):
        # one step of at most lr; the two clip coefficients agree to a few roundings, which m / sqrt(v) divides out but for eps:
        # 24 u of parameter and update on either side, and eps = 1e-8 against the clipped gradient's size, about 1e-5, times 8 u
        assert float((a - b).abs().max()) <= 2 * 24 * U * (float(b.abs().max()) + 1e-3)


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8bit"])
@pytest.mark.parametrize("strategy", ["supervised", "reinforcement"])
def test_trainer_epochs_and_checkpoint(dev, tmp_path, monkeypatch, optimizer, strategy):
    from src.common.config.config import Settings
    from src.gcn.train.trainer import Trainer
    shutil.copytree(os.path.join(GOLDEN, "datasets", "nsf_small"), tmp_path / "nsf_small")
    monkeypatch.setenv("GCN_UELB_MODEL_ROOT", str(tmp_path / "models"))
    monkeypatch.delenv("GCN_UELB_DATA_ROOT", raising=False)
    cfg = Settings(dict(data_root=str(tmp_path), dataset_name="nsf_small", num_train_data=12, batch_size=4, num_nodes=14, num_commodities=4,
                        voc_edges_in=3, voc_edges_out=2 if strategy == "supervised" else 1, hidden_dim=64, num_layers=2, mlp_layers=2,
                        aggregation="mean", learning_rate=1e-3, max_epochs=2, training_strategy=strategy, beam_size=2, seed=5,
                        optimizer=optimizer, max_grad_norm=1.0, rl_link_frequency_penalty=0.2))
    torch.manual_seed(0)
    tr = Trainer(cfg, torch.float32, torch.long)
    tr.train()
    assert len(tr.history) == 2 and all(np.isfinite(h[2]) for h in tr.history)
    assert float(tr.optimizer.grad_norm) > 0
    ckpt = torch.load(tmp_path / "models" / tr._get_model_filename(), weights_only=True)
    again = Trainer(cfg, torch.float32, torch.long)
    again.load_checkpoint(str(tmp_path / "models" / tr._get_model_filename()))
    again.optimizer.load_state_dict(ckpt["optimizer_state_dict"])
    p, q = next(iter(tr.optimizer.state)), next(iter(again.optimizer.state))
    assert torch.equal(tr.optimizer.state[p]["exp_avg"], again.optimizer.state[q]["exp_avg"])
    assert float(again.optimizer.state[q]["step"]) == 6
    assert any("exp_avg_exp" in st for st in again.optimizer.state.values()) == (optimizer == "adamw8bit")


class FixedScores(torch.nn.Module):
    def __init__(self, y):
        super().__init__()
        self.y = torch.nn.Parameter(y)

    def forward(self, x_edges, x_commodities, cap, x_nodes, y_edges=None, edge_cw=None, compute_loss=False, mask_invalid_edges=False):
        return self.y, None


def test_the_gradient_with_link_penalties_is_that_of_the_expected_reward(dev, monkeypatch):
    """Two routes, 0 - 1 - 3 and 0 - 2 - 3: the strategy's gradients of all four pairs (first draw, paths that count), weighted with the
    pairs' probabilities, add up to the derivative of the expected reward over both draws, taken by differences in double
    precision.  Without the first draw's probability the sum is another one (shown at the end)."""
    from src.gcn.algorithms.path_sampler import PathLogProbFn, PathSampler
    from src.gcn.training.reinforcement_strategy import ReinforcementLearningStrategy
    rho, presence, frequency = 1.4, 0.6, 0.3
    cfg = dict(rl_use_baseline=False, rl_normalize_advantages=False, rl_entropy_weight=0.0, rl_sampling_temperature=1.0, rl_sampling_top_p=1.0,
               rl_entropy_epsilon=0.0, rl_link_repetition_penalty=rho, rl_link_presence_penalty=presence, rl_link_frequency_penalty=frequency)
    cap = torch.zeros(1, 4, 4, device=dev)
    for i, j, c in ((0, 1, 10.0), (1, 3, 10.0), (0, 2, 3.0), (2, 3, 3.0)):
        cap[0, i, j] = c
    comm = torch.tensor([[[0, 3, 2]]], device=dev)
    path = {k: torch.tensor([[[0, k, 3] + [-1] * 7]], dtype=torch.int32, device=dev) for k in (1, 2)}
    length = torch.full((1, 1), 3, dtype=torch.int32, device=dev)
    y = torch.randn(1, 4, 4, 1, generator=torch.Generator().manual_seed(4))
    y[0, 0, 1, 0], y[0, 0, 2, 0] = 0.7, -0.4                                   # one of either sign
    data = dict(x_edges=None, x_commodities=comm[:, :, 2].float(), x_edges_capacity=cap, x_nodes=None, batch_commodities=comm)
    chosen = {}

    def forced(self):
        logp, paths, plen, *_ = PathLogProbFn.apply(self.y_pred_edges.float().contiguous(), self._cap, self._comm, float(self.temperature),
                                                    float(self.top_p), float(self.entropy_epsilon), None, (path[chosen["first"]], length))
        return paths, plen, logp
    monkeypatch.setattr(PathSampler, "draw_with_log_probs", forced)

    def probabilities(a):
        """p(first), p(second | first) in double precision from the scores of links 0 - 1 and 0 - 2."""
        def soft(z):
            e = np.exp(z - z.max())
            return e / e.sum()
        p, q = soft(a), np.empty((2, 2))
        for f in range(2):
            z = a.copy()
            z[f] = (z[f] / rho if z[f] > 0 else z[f] * rho) - presence - frequency
            q[f] = soft(z)
        return p, q

    at = np.array([float(y[0, 0, 1, 0]), float(y[0, 0, 2, 0])])
    p, q = probabilities(at)
    reward, total, size = {}, np.zeros(2), 0.0
    for f in (1, 2):
        for s in (1, 2):
            chosen["first"] = f
            strat = ReinforcementLearningStrategy(cfg)
            strat.replay_paths = (path[s], length)
            model = FixedScores(y.to(dev)).train()
            loss, m = strat.compute_loss(model, data, dev)
            loss.backward()
            assert not m["reinforce_fallback_used"]
            reward[s] = m["reward_individual"][0]
            grad = -model.y.grad.cpu().double().numpy()[0, :, :, 0]
            weight = p[f - 1] * q[f - 1, s - 1]
            total += weight * grad[0, 1:3]
            size += weight * np.abs(grad[0, 1:3]).max()
            grad[0, 1:3] = 0
            assert (grad == 0).all()                                            # the other nodes have one way on
    assert reward[1] != reward[2]

    def expected(a):
        p, q = probabilities(a)
        return sum(p[f] * q[f, s] * reward[s + 1] for f in range(2) for s in range(2))

    step, want = 1e-5, np.empty(2)
    for k in range(2):
        e = np.eye(2)[k] * step
        want[k] = (expected(at + e) - expected(at - e)) / (2 * step)
    # the fp32 softmax, its logarithm and the rules: about 20 roundings of each term; differences: step^2 and 1e-16 / step
    assert (np.abs(total - want) <= 64 * U * size + 1e-9).all(), (total, want)
    onehot = np.eye(2)
    first_term = sum(p[f] * q[f, s] * reward[s + 1] * (onehot[f] - p) for f in range(2) for s in range(2))
    assert np.abs(first_term).max() > 0.01


def test_draws_with_log_probabilities(dev):
    """The draw that draw() makes, with the log-probability and the gradient that evaluate() gives for its paths."""
    from src.gcn.algorithms.path_sampler import PathSampler
    from src.gcn.hip import lib as L
    B, V, C = 4, 14, 6
    cap, comm = graphs(B, V, C)
    kind = dict(temperature=1.3, top_p=0.9, entropy_epsilon=0.05)
    y = torch.randn(B, V, V, C, device=dev, generator=torch.Generator(dev).manual_seed(8)).requires_grad_()
    torch.manual_seed(21)
    L.reseed()
    paths, plen = PathSampler(y, cap, comm, **kind).draw()
    L.reseed()
    again, length, logp = PathSampler(y, cap, comm, **kind).draw_with_log_probs()
    assert torch.equal(paths, again) and torch.equal(plen, length) and logp.shape == (B,)
    _, want, _, _ = PathSampler(y, cap, comm, **kind).evaluate(paths, plen)
    assert torch.equal(logp, want)
    dy = torch.randn(B, device=dev)
    got, base = torch.autograd.grad(logp, [y], dy)[0], torch.autograd.grad(want, [y], dy)[0]
    assert float(base.abs().max()) > 0 and torch.equal(got, base)


@pytest.mark.parametrize("own, strategy, effective", [(0.01, 1.0, 0.01), (0.5, 0.02, 0.02), (0.01, 0.0, 0.01), (None, 0.02, 0.02), (None, 0.0, None)])
def test_the_smaller_of_two_clipping_norms_holds(dev, own, strategy, effective):
    """The optimizer's max_grad_norm and the strategy's: the first moment after one step is a tenth of the clipped gradient."""
    extra = dict(rl_grad_clip_max_norm=strategy, **({} if own is None else dict(max_grad_norm=own)))
    net, opt, strat, data = _strategy(dev, "adamw", **extra)
    params = list(net.parameters())
    grads = [torch.randn(p.shape, device=dev, generator=torch.Generator(dev).manual_seed(k)) for k, p in enumerate(params)]
    norm = float(torch.sqrt(sum((g.double() ** 2).sum() for g in grads)))
    assert strat.backward_step(sum((p * g).sum() for p, g in zip(params, grads)), opt, 1, 0)
    assert abs(strat.grad_norm_history[-1] - norm) <= 2e-6 * norm
    scale = 1.0 if effective is None else effective / (norm + 1e-6)
    for p, g in zip(params, grads):
        want = 0.1 * scale * g.double()
        # (1 - b1), the coefficient and two products: 8 roundings
        assert bool(((opt.state[p]["exp_avg"].double() - want).abs() <= 8 * U * want.abs() + 1e-44).all())
