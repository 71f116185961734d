"""CPU: the optional hidden parts of actor and critic (layer norm, gated feed-forward blocks, dropout)."""
import pytest
import torch
import yaml

from gsc_amd.agents import Batch, DDPGLearner
from gsc_amd.coordsim.reader import load_topology
from gsc_amd.models import Actor, GraphSet, MaskedInputMLP, QNetwork, count_params
from gsc_amd.parallel.dist import DistInfo
from gsc_amd.utils.checkpoint import load_actor, save_actor
from tests.conftest import cfg_path

ABILENE = cfg_path("networks", "abilene", "abilene-in4-rand-cap1-2.graphml")
TRIANGLE = cfg_path("networks", "triangle", "triangle-in1-cap10-delay10.graphml")


def _cfg(**kw):
    cfg = yaml.safe_load(open(cfg_path("config", "agent", "sample_agent_feedforward.yaml")))
    cfg["actor_hidden_layer_nodes"], cfg["critic_hidden_layer_nodes"] = [32], [24, 16]
    return {**cfg, **kw}


def _batch(B, seed=1, T=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)
    return Batch(r(B, 24, 3), torch.randint(0, T, (B,), generator=g), r(B, 1728), r(B) - 0.5, r(B, 24, 3),
                 (r(B) < 0.1).float())


def test_absent_options_leave_the_networks_as_they_were():
    cfg = yaml.safe_load(open(cfg_path("config", "agent", "sample_agent.yaml")))
    a, q = Actor(cfg, 3, 1728), QNetwork(cfg, 3, 1728)
    assert count_params(a) == 893628 and count_params(q) == 223997
    assert a.mlp.plain and q.mlp.plain and not list(a.buffers()) and not list(q.buffers())
    assert all(n.startswith(("embedder.", "mlp.layers.")) for n, _ in a.named_parameters())


def test_sizes_of_the_sample_config():
    cfg = yaml.safe_load(open(cfg_path("config", "agent", "sample_agent_feedforward.yaml")))
    block = lambda w: 2 * w + 2 * 4 * w * w + 8 * w + 4 * w * w + w      # norm, gate and up, down
    assert count_params(Actor(cfg, 3, 1728)) == 893628 + 2 * 256 + block(256)
    assert count_params(QNetwork(cfg, 3, 1728)) == 223997 + 2 * 64 + 2 * block(64)


def test_mask_folding_and_composed_projection_with_hidden_parts():
    """Folded == explicit concatenation, and critic(x, actor(x)) == the re-associated projection, values and gradients."""
    torch.manual_seed(3)
    cfg = _cfg()
    gs = GraphSet([load_topology(ABILENE), load_topology(TRIANGLE)], 24)
    masks = gs.action_masks(1, 3).double()
    q = QNetwork(cfg, 3, 1728).double().eval()
    emb, act = torch.randn(5, 22, dtype=torch.float64), torch.rand(5, 1728, dtype=torch.float64)
    tid = torch.tensor([0, 1, 0, 1, 1])
    torch.testing.assert_close(q.mlp(emb, tid, masks, act), q.mlp.forward_full(torch.cat([emb, masks[tid], act], 1)))
    one = GraphSet([load_topology(ABILENE)], 24)
    m1, t1 = one.action_masks(1, 3), torch.zeros(6, dtype=torch.long)
    actor, critic = Actor(cfg, 3, 1728).eval(), QNetwork(cfg, 3, 1728).eval()
    x = torch.rand(6, 24, 3)
    params = [p for p in [*actor.parameters(), *critic.parameters()]]
    q1 = critic(x, t1, one, m1, actor(x, t1, one, m1))
    q2 = critic.forward_on_actor(x, t1, one, m1, actor, actor.hidden(x, t1, one, m1))
    torch.testing.assert_close(q1, q2, rtol=1e-4, atol=1e-4)
    for a, b in zip(torch.autograd.grad(q1.sum(), params), torch.autograd.grad(q2.sum(), params)):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4)


def test_dropout_follows_mode_seed_step_and_site():
    torch.manual_seed(4)
    mlp = MaskedInputMLP(6, 0, 0, [40, 40], 3, blocks=2, dropout=0.5)
    x, t, m = torch.randn(50, 6), torch.zeros(50, dtype=torch.long), torch.zeros(1, 0)
    mlp.seed_dropout(5)
    run = lambda: mlp(x, t, m)
    mlp.eval()
    still = run()
    assert torch.equal(still, run())
    mlp.train()
    a = run()
    assert torch.equal(a, run()) and not torch.equal(a, still)
    mlp.advance_dropout()
    b = run()
    assert not torch.equal(a, b)
    mlp.drop_step.zero_()
    assert torch.equal(run(), a)
    mlp.seed_dropout(6)
    assert not torch.equal(run(), a)
    ones = torch.ones(64, 40)
    masks = [mlp._drop(ones, site) != 0 for site in (0, 1, -1, -2)]
    assert all(not torch.equal(p, q) for i, p in enumerate(masks) for q in masks[:i])
    mlp.eval()
    assert torch.equal(mlp._drop(ones, 0), ones) and torch.equal(mlp._drop(ones, 0, ones), 2 * ones)


def test_gradients_in_training_mode():
    """All parts together, dropout included, against differences (64 bits)."""
    torch.manual_seed(5)
    mlp = MaskedInputMLP(4, 3, 2, [6, 5], 2, norm=True, blocks=1, expansion=2, activation="gelu", dropout=0.3).double().train()
    x, extra = torch.randn(7, 4, dtype=torch.float64), torch.randn(7, 2, dtype=torch.float64)
    t, m = torch.randint(0, 2, (7,)), torch.rand(2, 3, dtype=torch.float64)
    params = dict(mlp.named_parameters())

    def f(x, *ps):
        return torch.func.functional_call(mlp, dict(zip(params, ps)), (x, t, m, extra))

    assert torch.autograd.gradcheck(f, (x.requires_grad_(), *[p.detach().requires_grad_() for p in params.values()]))


@pytest.mark.parametrize("key,value", [("hidden_layer_norm", "batch"), ("feedforward_blocks", -1), ("feedforward_blocks", 1.5),
                                       ("feedforward_expansion", 0), ("feedforward_activation", "relu"), ("dropout", 1.0),
                                       ("dropout", -0.1), ("hidden_layer_nodes", [])])
@pytest.mark.parametrize("net,cls", [("actor", Actor), ("critic", QNetwork)])
def test_refused_options(net, cls, key, value):
    with pytest.raises(ValueError):
        cls(_cfg(**{f"{net}_{key}": value}), 3, 1728)


def test_learner_updates_every_part_and_resumes(tmp_path):
    cfg = _cfg(actor_dropout=0.1, critic_dropout=0.2, learning_rate=1e-3)
    gs = GraphSet([load_topology(ABILENE)], 24, "cpu")
    make = lambda: DDPGLearner(cfg, 3, 1728, gs, 1, 3, "cpu", seed=3)
    L = make()
    assert not L.native_ok and not L.actor.training and not L.critic.training
    before = [fp.flat.clone() for fp in (L.actor_flat, L.critic_flat)]
    for k in range(3):
        L.update(_batch(16, seed=k))
    for fp, old in zip((L.actor_flat, L.critic_flat), before):
        for name, p, o in zip(fp.names, fp.params, fp.offsets):
            assert (fp.flat[o:o + p.numel()] != old[o:o + p.numel()]).any(), name
    assert int(L.critic.mlp.drop_step) == int(L.actor.mlp.drop_step) == 3
    assert not L.actor.training and not L.critic.training
    # a resumed learner continues exactly, its masks included
    R = make()
    R.load_state_dict(L.state_dict())
    for a in (L, R):
        a.update(_batch(16, seed=9))
    for name in ("actor_flat", "critic_flat", "target_actor_flat", "target_critic_flat"):
        assert torch.equal(getattr(L, name).flat, getattr(R, name).flat)
    save_actor(str(tmp_path / "a.pt"), L.actor, cfg, 3, 1728, 24, 1, 3)
    actor, _ = load_actor(str(tmp_path / "a.pt"))
    b = _batch(4)
    with torch.no_grad():
        torch.testing.assert_close(actor(b.obs, b.topo, gs, L.masks), L.act(b.obs, b.topo), rtol=0, atol=0)


def test_every_rank_draws_its_own_masks():
    cfg = _cfg(actor_dropout=0.1, critic_dropout=0.2)
    gs = GraphSet([load_topology(ABILENE)], 24, "cpu")
    a, b = (DDPGLearner(cfg, 3, 1728, gs, 1, 3, "cpu", DistInfo(rank=r), seed=3) for r in (0, 1))
    assert torch.equal(a.critic_flat.flat, b.critic_flat.flat)
    assert len({n.mlp.drop_seed for L in (a, b) for n in (L.actor, L.critic)}) == 4


def test_renewed_parameters_keep_storage_and_places():
    L = DDPGLearner(_cfg(), 3, 1728, GraphSet([load_topology(ABILENE)], 24, "cpu"), 1, 3, "cpu", seed=3)
    old = list(L.critic_flat.params)
    L.critic_flat.renew_parameters()
    new = dict(L.critic.named_parameters())
    for name, p, q in zip(L.critic_flat.names, old, L.critic_flat.params):
        assert new[name] is q and q is not p and q.data_ptr() == p.data_ptr() and q.requires_grad
    L.update(_batch(8))
    assert all(torch.equal(p, q) for p, q in zip(old, L.critic_flat.params))
