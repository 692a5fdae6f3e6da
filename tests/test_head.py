"""The gated classifier head on the CPU: formula, options, checkpoints, entry scripts."""
import sys

import pytest
import torch

import ffn_oracle as oracle
from ddl.config import parse_config
from ddl.models import HeadConfig, create_stage
from ddl.models.head import PARAMS, GatedHead

from test_entrypoints import SMALL, _env, _run, _torchrun

CFG = HeadConfig("gated", width=48, dropout=0.25)


def block64(m, f, keep):
    """The block in 64 bits; keep: the scaled dropout mask."""
    p = {n: t.double() for n, t in m.state_dict().items()}
    h = oracle.norm(f, p["norm_in.weight"], p["norm_in.bias"], "layer", 1e-5)
    y = oracle.linear(oracle.gated(h, p["gate.weight"], p["up.weight"], p["gate.bias"], p["up.bias"]), p["down.weight"], p["down.bias"])
    return oracle.norm(f + p["scale"] * y * keep, p["norm_out.weight"], p["norm_out.bias"], "layer", 1e-5)


def test_gated_head_formula():
    torch.manual_seed(0)
    m = GatedHead(40, CFG)
    assert set(PARAMS) == {n for n, _ in m.named_parameters()}
    f = torch.randn(6, 40)
    m.eval()
    # values below 8, four fp32 stages of at most 64 terms each: 4 * 80 * 2^-24 * 8
    assert (m(f).double() - block64(m, f.double(), 1.0)).abs().max() < 1.6e-4
    m.train()
    key = m.rng("cpu").state.tolist()
    keep = torch.from_numpy(oracle.kept(key, 240, 0.25)).double().view(6, 40) / 0.75
    assert (m(f).double() - block64(m, f.double(), keep)).abs().max() < 1.6e-4
    assert m.rng("cpu").state.tolist() == [key[0], key[1] + 1]
    m(f).sum().backward()
    assert all(p.grad is not None for p in m.parameters())


def test_options():
    cfg = parse_config("single", ["--head", "gated", "--head-width", "96", "--head-dropout", "0.3"])
    assert cfg.head_config() == HeadConfig("gated", 96, 0.3)
    assert parse_config("single", []).head_config() == HeadConfig()
    for bad in (dict(kind="mlp"), dict(width=0), dict(dropout=1.0), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            HeadConfig(**bad)


def test_default_head_is_unchanged_and_backbones_interchange(tmp_path):
    torch.manual_seed(0)
    plain = create_stage(("head",), "cpu", 5)
    assert [n for n, _ in plain.named_parameters()] == ["features.norm5.weight", "features.norm5.bias", "classifier.weight",
                                                       "classifier.bias"]
    torch.save(plain.state_dict(), tmp_path / "plain.pt")
    gated = create_stage(("head",), "cpu", 5, pretrained=str(tmp_path / "plain.pt"), head=CFG)
    assert {n for n in gated.state_dict() if n.startswith("ffn.")} == {"ffn." + n for n in PARAMS}
    for n, t in plain.state_dict().items():
        assert torch.equal(gated.state_dict()[n], t)
    x = torch.randn(2, 1024, 3, 3)
    assert gated.eval()(x).shape == (2, 5)


def test_entry_scripts_train_with_the_gated_head(tmp_path):
    env = _env(tmp_path)
    head = ["--head", "gated", "--head-width", "64"]
    out = _run([sys.executable, "single.py", *SMALL, "--batch-size", "8", "--save-every", "1", *head], env)
    assert "Epoch 0 | Training Accuracy" in out
    out = _run([sys.executable, "single.py", *SMALL[2:], "--epochs", "2", "--batch-size", "8", "--snapshot-job-id", "job-123",
                "--snapshot-epoch", "0", *head], env)
    assert "Resuming training from snapshot at Epoch 1" in out
    _torchrun(2, "pp.py", [*SMALL, "--batch-size", "10", *head], env)


def test_dropout_keys_move_with_the_head():
    m = GatedHead(40, CFG)
    m.train()
    m(torch.randn(6, 40))
    key = m.rng("cpu").state.tolist()
    assert m.rng(torch.device("meta")).state.device.type == "meta"
    m._rng.state = torch.tensor(key)
    assert m.rng("cpu").state.tolist() == key and key[1] == 1


def test_a_resumed_run_draws_the_masks_of_the_uninterrupted_one(tmp_dirs):
    """Two epochs in one go, and with a stop between them: the same losses and parameters, bit for bit."""
    from ddl.cli import run_training
    args = [*SMALL[2:], "--batch-size", "8", "--seed", "5", "--head", "gated", "--head-width", "64", "--head-dropout", "0.5"]
    whole = run_training("single", [*args, "--epochs", "2", "--save-every", "1"])
    first = run_training("single", [*args, "--epochs", "1", "--save-every", "1"])
    assert first.history[0]["loss"] == whole.history[0]["loss"]
    second = run_training("single", [*args, "--epochs", "2", "--snapshot-job-id", first.job_id, "--snapshot-epoch", "0"])
    assert second.history[0]["epoch"] == 1 and second.history[0]["loss"] == whole.history[1]["loss"]
    a, b = whole.s.model.state_dict(), second.s.model.state_dict()
    assert all(torch.equal(a[n], b[n]) for n in a)
    key = second.s.model.ffn.rng("cpu").state[1].item()
    assert key == (1 << 32) + 2                                       # two steps of the second epoch


def test_seek():
    from ddl import ops
    rng = ops.DropoutRng(7, "cpu", stream=3)
    rng.seek(5)
    assert rng.next_key().tolist() == [7, (3 << 48) + 5] and rng.next_key().tolist() == [7, (3 << 48) + 6]
    for bad in (-1, 2 ** 48):
        with pytest.raises(ValueError):
            rng.seek(bad)
