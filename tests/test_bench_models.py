"""bench.py names the networks that it runs (CPU, tiny sizes)."""
from tests.test_bench_contract import _run


def test_model_of_an_agent_config():
    sizes = ("--envs", "2", "--batch-size", "8", "--steps", "1", "--warmup", "1")
    own = _run(*sizes, "--agent-config", "configs/config/agent/sample_agent_feedforward.yaml")["config"]["model"]
    block = lambda w: 2 * w + 2 * 4 * w * w + 8 * w + 4 * w * w + w      # norm, gate and up, down
    assert f"actor {893628 + 2 * 256 + block(256):,} params" in own
    assert f"critic {223997 + 2 * 64 + 2 * block(64):,} params" in own and "sample_agent_feedforward.yaml" in own
    assert "actor [256] 893,628 params, critic [64] 223,997 params" in _run(*sizes)["config"]["model"]
