"""Training with this package's operators (TrainConfig.hip_ops) twice from one seed: every sum of
theirs has a fixed order, and so have the step's others at this size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["span", "copy"])
def test_two_runs_give_the_same_weights(fmt):
    from smsgate_amd.models.train import TrainConfig, train_extractor

    cfg = TrainConfig(model="small", steps=6, batch=16, n_examples=200, warmup=2, log_every=0, answer_format=fmt,
                      hip_ops=True, ema=0.0)
    a, b = (train_extractor(cfg, device="cuda", log=lambda *_: None) for _ in range(2))
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert torch.equal(p, q), n
