"""GPU: actor and critic with layer norm, gated feed-forward blocks and dropout, in the learner and the trainer."""
import pytest
import torch
import yaml

from gsc_amd.agents import DDPGLearner
from gsc_amd.coordsim.reader import load_topology
from gsc_amd.models import GraphSet, MaskedInputMLP
from tests.conftest import cfg_path
from tests.feedforward_bounds import U
from tests.test_gpu_graphs import _batches

pytestmark = pytest.mark.gpu

ABILENE = cfg_path("networks", "abilene", "abilene-in4-rand-cap1-2.graphml")


def _cfg(**kw):
    cfg = yaml.safe_load(open(cfg_path("config", "agent", "sample_agent_feedforward.yaml")))
    return {**cfg, **kw}


def _learner(cfg, seed=5, **kw):
    return DDPGLearner(cfg, 3, 1728, GraphSet([load_topology(ABILENE)], 24, "cuda"), 1, 3, "cuda", seed=seed, **kw)


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("sizes", [(1, [40]), (33, [64, 48]), (700, [256])])
def test_network_gradients_against_64_bits(sizes, autocast):
    """The whole MLP in training mode on the GPU against the same module in 64 bits on the CPU (same masks)."""
    B, hidden = sizes
    torch.manual_seed(B)
    ref = MaskedInputMLP(22, 60, 30, hidden, 7, norm=True, blocks=2, dropout=0.25).train()
    gpu = MaskedInputMLP(22, 60, 30, hidden, 7, norm=True, blocks=2, dropout=0.25).train()
    gpu.load_state_dict(ref.state_dict())
    gpu.cuda()
    ref.double()
    for m in (ref, gpu):
        m.seed_dropout(77)
        m.advance_dropout()
    g = torch.Generator().manual_seed(B)
    x, extra, masks = torch.randn(B, 22, generator=g), torch.rand(B, 30, generator=g), torch.rand(2, 60, generator=g).round()
    topo, dy = torch.randint(0, 2, (B,), generator=g), torch.randn(B, 7, generator=g)
    want_y = ref(x.double(), topo, masks.double(), extra.double())
    want = torch.autograd.grad(want_y, list(ref.parameters()), dy.double())
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        y = gpu(x.cuda(), topo.cuda(), masks.cuda(), extra.cuda())
        got = torch.autograd.grad(y, list(gpu.parameters()), dy.cuda().to(y.dtype))
    # roundings on the longest path there and back: in fp32 about 8 w + 100 of U (sums of up to 4 w terms), in bf16 about
    # 40 of 2^-8, adding like independent errors (sqrt(40)); relu flips where a pre-activation is within its error of 0
    # (a share 2 e of the elements, each an error of its own size: sqrt(2 e) relative); gains up to 4
    e = 2.0 ** -8 * 40 ** 0.5 if autocast else (8 * hidden[-1] + 100) * U
    tol = 4 * (e + (2 * e / 40 ** 0.5) ** 0.5)
    assert (y.cpu().double() - want_y).norm() <= tol * want_y.norm()
    scale = max(b.norm().item() / b.numel() ** 0.5 for b in want)
    for (n, _), a, b in zip(ref.named_parameters(), got, want):
        assert (a.cpu().double() - b).norm() <= tol * (b.norm() + scale * b.numel() ** 0.5), n


@pytest.mark.parametrize("B", [512, 9000])
def test_graphed_updates_equal_eager_ones(B):
    """Updates replayed from one captured graph == eager updates, dropout masks included, with eager work between the
    replays and an eager graph of the same parameters alive during the capture."""
    cfg = _cfg(actor_dropout=0.1, critic_dropout=0.2)
    eager, graphed = _learner(cfg), _learner(cfg)
    assert not eager.native_ok
    static = type(_batches(1, B, "cuda")[0])(*(torch.empty_like(t) for t in _batches(1, B, "cuda")[0]))
    alive = None
    for k, b in enumerate(_batches(7, B, "cuda")):
        eager.update(b)
        for d, s in zip(static, b):
            d.copy_(s)
        if k == 2:   # the next call captures
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                alive = graphed.critic(b.obs, b.topo, graphed.graphs, graphed.masks, b.actions)
        graphed.update_graphed(static, warmup=2)
        for name in ("actor_flat", "critic_flat", "target_actor_flat", "target_critic_flat"):
            assert torch.equal(getattr(graphed, name).flat, getattr(eager, name).flat), (k, name)
        assert torch.equal(graphed.act(b.obs, b.topo), eager.act(b.obs, b.topo))
    assert graphed._graphs is not None and graphed.updates == 7 and int(graphed.critic.mlp.drop_step) == 7
    assert alive.isfinite().all()


def test_trainer_runs_with_the_sample_config():
    """Batched trainer on the device simulator with the sample configuration: acting, replay and updates, graphed."""
    from gsc_amd.agents import BatchedTrainer, TrainerConfig
    from gsc_amd.sim.batched import load_batched_from_paths
    cfg = _cfg()
    sim = load_batched_from_paths([ABILENE], cfg_path("service_functions", "abc.yaml"),
                                  cfg_path("config", "simulator", "sample_config.yaml"), cfg, 8, device="cuda")
    tr = BatchedTrainer(cfg, sim, TrainerConfig(num_envs=8, batch_size=64, learning_starts=1))
    before = tr.learner.actor_flat.flat.clone()
    for _ in range(6):
        tr.step()
    m = tr.metrics()
    torch.cuda.synchronize()
    sim.check_flags()
    assert all(v == v for k, v in m.items() if k != "mean_episode_return"), m
    assert (tr.learner.actor_flat.flat != before).any() and tr.learner.actor_flat.flat.isfinite().all()
    assert int(tr.learner.critic.mlp.drop_step) == tr.learner.updates
