"""The Muon operators after a bounded wait of some native kernel has run out: the host sets the
device's status word, as a kernel that gives up does."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(64, 48), (300, 200), (200, 310), (20, 12)]  # single-CTA and whole-GPU matrices


@pytest.fixture
def status():
    from synthefy_nori_b200 import ops

    word = ops.status_word(torch.device("cuda"))
    word.fill_(7)
    yield word
    word.zero_()


def _buffers():
    torch.manual_seed(0)
    n = sum(r * c for r, c in SHAPES)
    offsets = [sum(r * c for r, c in SHAPES[:i]) for i in range(len(SHAPES))]
    return offsets, [torch.randn(n, device="cuda") for _ in range(4)]


def test_muon_step_leaves_every_buffer(status):
    from synthefy_nori_b200 import ops

    offsets, (data, grad, mom, ema) = _buffers()
    plan = ops.MuonPlan(SHAPES, offsets, "cuda")
    before = [t.clone() for t in (data, grad, mom, ema)]
    for nesterov in (True, False):
        ops.muon_step(plan, data, grad, mom, lr=0.1, nesterov=nesterov, ema=ema)
    assert all(torch.equal(a, b) for a, b in zip(before, (data, grad, mom, ema)))
    with pytest.raises(RuntimeError, match="timeout"):
        ops.check_status(data.device)
    status.zero_()
    ops.muon_step(plan, data, grad, mom, lr=0.1, ema=ema)
    assert not any(torch.equal(a, b) for a, b in zip((before[0], *before[2:]), (data, mom, ema)))


def test_newton_schulz_leaves_its_output(status):
    from synthefy_nori_b200 import ops

    for shape in SHAPES:
        g, out = torch.randn(2, *shape, device="cuda"), torch.full((2, *shape), 3.0, device="cuda")
        ops.newton_schulz(g, out=out)
        assert (out == 3.0).all()


def test_trainer_raises_where_it_reads_its_counters(status):
    from synthefy_nori_b200.models.config import preset_config
    from synthefy_nori_b200.training.trainer import NoriTrainer, TrainConfig
    from synthefy_nori_b200.utils.loading import build_model

    torch.manual_seed(0)
    tr = NoriTrainer(build_model(preset_config("nori-tiny")), TrainConfig(optimizer="muon"), torch.device("cuda", 0))
    with pytest.raises(RuntimeError, match="timeout"):
        tr.poll()
    status.zero_()
    assert tr.poll()["skipped_steps"] == 0
    tr.close()
