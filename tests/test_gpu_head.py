"""The gated classifier head in the native engine (models/head.py, csrc/ffn_*.hip)."""
import pytest
import torch

import ffn_oracle as oracle
from test_head import block64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from ddl import ops
    ops.require_ext()
    return torch.device("cuda", 0)


def _stages(dev, dropout):
    """The native head unit and its 64-bit twin with the same weights."""
    from ddl.models import HeadConfig, create_stage
    from ddl.models.densenet import DenseNetStage
    torch.manual_seed(3)
    cfg = HeadConfig("gated", width=200, dropout=dropout)
    native = create_stage(("head",), dev, 5, head=cfg)
    with torch.no_grad():
        for n, p in native.named_parameters():
            if n.startswith("ffn.") or n.startswith("classifier."):
                p.add_(0.1 * torch.randn_like(p))
    plain = DenseNetStage(("head",), 5, cfg)
    plain.load_state_dict({k: v.cpu() for k, v in native.export_state_dict().items()})
    return native, plain.double().to(dev)


def _forward64(plain, x, keep):
    """logits of the twin, with a given scaled dropout mask"""
    f = torch.relu(plain.features(x)).mean((2, 3))
    p = dict(plain.ffn.named_parameters())
    h = oracle.norm(f, p["norm_in.weight"], p["norm_in.bias"], "layer", 1e-5)
    y = oracle.linear(oracle.gated(h, p["gate.weight"], p["up.weight"], p["gate.bias"], p["up.bias"]), p["down.weight"], p["down.bias"])
    return plain.classifier(oracle.norm(f + p["scale"] * y * keep, p["norm_out.weight"], p["norm_out.bias"], "layer", 1e-5))


@pytest.mark.parametrize("B", [1, 6, 40])
@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_head_unit_against_64_bits(dev, B, dropout):
    native, plain = _stages(dev, dropout)
    native.train(), plain.train()
    x = torch.randn(B, 7, 7, 1024, generator=torch.Generator().manual_seed(B)).to(dev)
    d = torch.randn(B, 5, generator=torch.Generator().manual_seed(B + 1)).to(dev)
    keep = 1.0
    if dropout:
        key = native._dropout_rngs[0].state.tolist()
        keep = torch.from_numpy(oracle.kept(key, B * 1024, dropout)).to(dev).double().view(B, 1024) / (1 - dropout)
    xn, xp = x.clone().requires_grad_(True), x.double().permute(0, 3, 1, 2).contiguous().requires_grad_(True)
    got = native(xn)
    want = _forward64(plain, xp, keep)
    # values of order one through five fp32 stages of up to 1024 terms: relative 2e-5 of the largest value each
    scale = want.abs().max().item()
    assert (got.double() - want).abs().max() <= 1e-4 * scale
    got.backward(d)
    want.backward(d.double())
    for n, p in native.named_parameters():
        w = dict(plain.named_parameters())[n].grad
        assert (p.grad.double() - w).abs().max() <= 2e-4 * w.abs().max() + 1e-6, n
    w = xp.grad.permute(0, 2, 3, 1)
    assert (xn.grad.double() - w).abs().max() <= 2e-3 * w.abs().max()
    # a second backward adds to the gradients
    once = native.arena.flat_grad.clone()
    if not dropout:
        native(x.clone().requires_grad_(True)).backward(d)
        torch.testing.assert_close(native.arena.flat_grad, 2 * once, rtol=1e-5, atol=1e-6)
        plain.features(xp)                                           # the twin's running statistics follow
    native.eval(), plain.eval()
    with torch.no_grad():
        got, again, want = native(x), native(x), _forward64(plain, xp, 1.0)
    assert torch.equal(got, again) and (got.double() - want).abs().max() <= 1e-4 * want.abs().max()


def test_graphed_training_draws_new_masks_and_matches_eager(dev):
    """Five steps of the trainer's captured step against the same steps launched eagerly: the device-side counter advances with every
    replay, so both draw the same masks and end in the same parameters, bit for bit."""
    from ddl import comm
    from ddl.config import TrainConfig
    from ddl.trainer import SingleStrategy
    ctx = comm.CommContext(0, 1, 0, dev, "none")
    finals = []
    for graph in (True, False):
        torch.manual_seed(11)
        cfg = TrainConfig(strategy="single", batch_size=6, image_size=64, hip_graph=graph, head="gated", head_width=256, head_dropout=0.5)
        strat = SingleStrategy(cfg, ctx)
        strat.model.train()
        g = torch.Generator().manual_seed(0)
        losses = []
        for _ in range(6):
            x = torch.randint(0, 256, (6, 3, 64, 64), dtype=torch.uint8, generator=g).to(dev)
            y = torch.randint(0, 5, (6,), generator=g).to(dev)
            losses.append(float(strat.train_step(x, y, 6)[0].detach()))
        torch.cuda.synchronize()
        calls = int(strat.model._dropout_rngs[0].state[1])
        finals.append((losses, strat.arena.flat_param.clone(), calls))
    assert finals[0][2] == finals[1][2] == 6
    assert finals[0][0] == finals[1][0] and torch.equal(finals[0][1], finals[1][1])


@pytest.mark.parametrize("fwd_lanes", [1, 2])
def test_pipeline_lanes_draw_the_serial_masks(dev, fwd_lanes):
    """Concurrent micro-batches of one stage: the graphed run against --debug-sync (one stream, eager), bit for bit."""
    from ddl import comm
    from ddl.config import TrainConfig
    from ddl.trainer import build_strategy
    ctx = comm.CommContext(0, 1, 0, dev, "none")
    finals = []
    for graph, debug in ((True, False), (False, True)):
        torch.manual_seed(5)
        cfg = TrainConfig(strategy="pp", batch_size=10, num_microbatches=5, image_size=64, hip_graph=graph, debug_sync=debug, pp_lanes=2,
                          pp_fwd_lanes=fwd_lanes, split_points=[], head="gated", head_width=128, head_dropout=0.5)
        strat = build_strategy(cfg, ctx)
        strat.model.train()
        g = torch.Generator().manual_seed(100)
        losses = []
        for _ in range(5):
            x = torch.randint(0, 256, (10, 3, 64, 64), dtype=torch.uint8, generator=g).to(dev)
            y = torch.randint(0, 5, (10,), generator=g).to(dev)
            losses.append(float(strat.train_step(x, y, 10)[0].detach()))
        torch.cuda.synchronize()
        finals.append((losses, strat.arena.flat_param.clone()))
    assert finals[0][0] == finals[1][0] and torch.equal(finals[0][1], finals[1][1])


def test_evaluation_keeps_nothing_for_a_backward_pass(dev):
    """Without gradients neither the projections' fp32 sums nor the norms' statistics are written; the logits are the same."""
    from ddl.models import head
    native, _ = _stages(dev, 0.2)
    native.eval()
    B, width, made = 40, 200, {}
    x = torch.randn(B, 7, 7, 1024, generator=torch.Generator().manual_seed(1)).to(dev)

    def run(grad):
        with torch.set_grad_enabled(grad):
            before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
            y = native(x)
            return y.detach(), torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before

    run(False)
    (a, plain), (b, kept) = run(False), run(True)
    assert torch.equal(a, b)
    assert kept - plain >= 2 * B * width * 4 + 2 * 4 * B * 4          # two planes of sums, the statistics of two norms
    ext = head.ops.require_ext()
    unit = native.unit_objs[-1]
    f = torch.randn(B, 1024, generator=torch.Generator().manual_seed(2)).to(dev)
    h, saved = head.native_forward(ext, unit.ffn, f, 0.0, None, False)
    again, _ = head.native_forward(ext, unit.ffn, f, 0.0, None, True)
    assert torch.equal(h, again) and [t is None for t in saved] == [False, False, True, True, False, False, True]


def test_portable_head_moves_between_devices(dev):
    """A step on the CPU, then .to(GPU): the next step draws the next mask there."""
    from ddl.models import HeadConfig
    from ddl.models.head import GatedHead
    torch.manual_seed(4)
    m = GatedHead(40, HeadConfig("gated", width=48, dropout=0.25))
    f = torch.randn(6, 40)
    m(f)
    state = m.rng("cpu").state.tolist()
    m.to(dev)
    got = m(f.to(dev))
    keep = torch.from_numpy(oracle.kept(state, 240, 0.25)).double().view(6, 40) / 0.75
    assert (got.cpu().double() - block64(m.cpu(), f.double(), keep)).abs().max() < 1.6e-4       # the bound of tests/test_head.py
    assert m.rng(dev).state.tolist() == [state[0], state[1] + 1]


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_masks_follow_the_epoch(dev, graph):
    """The keys of an epoch do not depend on how many steps ran before it, in a captured step either."""
    from ddl import comm
    from ddl.config import TrainConfig
    from ddl.trainer import SingleStrategy
    ctx = comm.CommContext(0, 1, 0, dev, "none")
    torch.manual_seed(11)
    strat = SingleStrategy(TrainConfig(strategy="single", batch_size=6, image_size=64, hip_graph=graph, head="gated", head_width=64,
                                       head_dropout=0.5), ctx)
    strat.model.train()
    x = torch.randint(0, 256, (6, 3, 64, 64), dtype=torch.uint8, generator=torch.Generator().manual_seed(0)).to(dev)
    y = torch.randint(0, 5, (6,), generator=torch.Generator().manual_seed(1)).to(dev)
    for epoch, steps in ((0, 3), (1, 2), (4, 1)):
        strat.model.set_epoch(epoch)
        for _ in range(steps):
            strat.train_step(x, y, 6)
        torch.cuda.synchronize()
        assert strat.model._dropout_rngs[0].state[1].item() == (epoch << 32) + steps
    strat.model.ensure_buffer_lanes(1)
    assert strat.model._dropout_rngs[1].state[1].item() == (1 << 48) + (4 << 32)
