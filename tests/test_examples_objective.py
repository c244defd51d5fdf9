"""The RL weight-sync example with a loss for its step: on CPU (gloo) ranks every
rank's log-probabilities agree to the last bit and the weights arrive exactly;
the step's gradient is the formula's."""
import pytest
import torch

from tests import _losses as oracle
from tests._mp import run_ranks


def _worker(rank, world, objective):
    from results_b200.examples import rl_weight_sync

    return rl_weight_sync.main(["--device", "cpu", "--small", "--layers", "1", "--steps", "3", "--objective", objective])


@pytest.mark.parametrize("objective", ["policy", "preference", "distill"])
def test_example_runs(objective):
    assert run_ranks(_worker, 2, args=(objective,)) == [True, True]


def _check_gradients(device, rel):
    from results_b200.examples import rl_weight_sync as ex
    from results_b200.models.shapes import glm4_9b_specs, make_state_dict

    specs = glm4_9b_specs(layers=1, hidden=64, heads=2, kv_heads=1, head_dim=32, ffn=64, vocab=500)
    sd = make_state_dict(specs, seed=1, device=device, dtype=torch.float32)
    hidden, actions = ex.rollout(sd, 5)
    old = ex.score(sd, hidden, actions)
    logits = hidden @ sd["lm_head.weight"].t()
    g = torch.Generator().manual_seed(1005)
    for objective in ("policy", "preference", "distill"):
        if objective == "policy":
            adv = torch.randn(32, generator=g).to(device)
            want = oracle.policy(logits, actions, old, adv, old, None, 0.2, 0.2, 0.05, 1.0, None)
        elif objective == "preference":
            want = oracle.preference(logits, actions, old.view(8, 4).sum(1), list(range(0, 33, 4)), 0.1, 0.0, False, 1.0)
        else:
            g = torch.Generator().manual_seed(1005)
            top = (logits.float() + torch.randn(logits.shape, generator=g).to(device)).topk(16)
            want = oracle.distill(logits, top.indices, top.values, None, 1.0, None)
        loss, grad = ex.objective_step(sd, objective, 5, hidden, actions, old)
        assert abs(float(loss) - float(want["loss"])) <= rel * (1 + abs(float(want["loss"])))
        ref = want["grad"].t() @ hidden.double()
        # 32 terms a sum, each product and sum rounded to fp32, the logits' gradient within rel of the slope
        off = want["slope"].abs()[:, None].expand_as(want["grad"]).t() @ hidden.double().abs()
        assert torch.all((grad.double() - ref).abs() <= (rel + 34 * 2.0 ** -24) * off)


def test_example_gradients():
    _check_gradients("cpu", 2.0 ** -20)


@pytest.mark.gpu
def test_example_gradients_gpu():
    # a row's sum takes a thread 500 / 256 additions and 64 joins, its slope carries that over: below 128 half steps
    assert not torch.backends.cuda.matmul.allow_tf32
    _check_gradients("cuda", 2.0 ** -17)
