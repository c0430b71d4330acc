"""A network with the norms around its residual blocks, trained the way a user trains it: forward, physics loss, backward, clipping and Adam
over its separate parameters, through the operators one after the other and through Trainer(engine="autograd")."""
import pytest
import torch
from torch.utils.data import DataLoader

import block_norm_ref as ref
from fluidnet_amd.config.training_config import PhysicsLossConfig, TrainingConfig
from fluidnet_amd.models.block_norm import GatedResidual, PreNorm
from fluidnet_amd.models.unet import UNetConfig
from fluidnet_amd.training.grad_clip import clip_grad_norm_
from fluidnet_amd.training.optim import ClipAdam
from fluidnet_amd.training.trainer import Trainer

pytestmark = pytest.mark.gpu
C = 40


class PixelNet(torch.nn.Module):
    """[B,6,H,W] -> [B,3,H,W], channels last inside: a projection, two blocks (a linear map each, over tokens), a projection."""
    model_name = "PixelNet"

    def __init__(self, dtype=torch.float32):
        super().__init__()
        self.stem, self.head = torch.nn.Linear(6, C), torch.nn.Linear(C, 3)
        self.first = PreNorm(C, kind="layer", bias=True)
        self.blocks = torch.nn.ModuleList(torch.nn.Linear(C, C) for _ in range(2))
        self.gates = torch.nn.Linear(C, C)
        self.joins = torch.nn.ModuleList([GatedResidual(C, kind="layer", bias=True, scale_init=0.5, gate_act="sigmoid"),
                                          GatedResidual(C, kind="rms", post=False, channel_gate=0.3, gate_act="tanh")])
        self.to(dtype)

    def forward(self, x):
        x = self.stem(x.permute(0, 2, 3, 1).to(self.stem.weight.dtype))
        h = self.first(x)
        x, h = self.joins[0](x, self.blocks[0](h), self.gates(h))
        x, h = self.joins[1](x, self.blocks[1](h))
        return self.head(h).permute(0, 3, 1, 2).float()


def _same_in_64_bits(net, x, weight):
    """The loss sum(weight * net(x)) and its gradients, by torch alone in 64 bits on the CPU."""
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in net.named_parameters()}
    lin = lambda n, v: v @ p[n + ".weight"].t() + p[n + ".bias"]  # noqa: E731
    v = lin("stem", x.cpu().double().permute(0, 2, 3, 1))
    _, h = ref.forward({"x": v, "post": False, "pre": True, "pre_weight": p["first.weight"], "pre_bias": p["first.bias"]}, "layer", "identity", 1.0, 1e-6)
    j = lambda k, *names: {n: p[f"joins.{k}.{n}"] for n in names}  # noqa: E731
    v, h = ref.forward({"x": v, "branch": lin("blocks.0", h), "gate": lin("gates", h), "post": True, "pre": True,
                        **j(0, "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")}, "layer", "sigmoid", 1.0, 1e-6)
    v, h = ref.forward({"x": v, "branch": lin("blocks.1", h), "post": False, "pre": True, **j(1, "gate", "pre_weight")}, "rms", "tanh", 1.0, 1e-6)
    loss = (lin("head", h).permute(0, 3, 1, 2) * weight.cpu().double()).sum()
    return float(loss.detach()), dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def test_gradients_clip_and_step_together():
    """Some 600 32-bit operations lie on the longest path (two products over 40 channels, three norms, their backward, sums over 200 rows),
    each good for 2^-24; normalising rows whose values reach four deviations grows errors fivefold: 2e-4 of a gradient's norm."""
    torch.manual_seed(1)
    net = PixelNet().cuda()
    x, weight = torch.randn(2, 6, 10, 10, device="cuda"), torch.randn(2, 3, 10, 10, device="cuda")
    want, grads = _same_in_64_bits(net, x, weight)
    opt, start = ClipAdam(net.parameters(), 1e-2, max_norm=None), {k: v.detach().cpu().double() for k, v in net.named_parameters()}
    loss = (net(x) * weight).sum()
    loss.backward()
    assert abs(float(loss.detach()) - want) < 2e-4 * abs(want) + 1e-2
    for k, p in net.named_parameters():
        assert float((p.grad.cpu().double() - grads[k]).norm()) < 2e-4 * float(grads[k].norm()) + 1e-6, k
    norm = clip_grad_norm_(net.parameters(), 1.0)
    total = float(torch.cat([g.reshape(-1) for g in grads.values()]).norm())
    assert abs(float(norm) - total) < 2e-4 * total
    opt.step()
    for k, p in net.named_parameters():                        # a first step is lr * g / (|g| + eps) of the clipped gradient
        g = p.grad.cpu().double()
        assert torch.allclose(p.detach().cpu().double(), start[k] - 1e-2 * g / (g.abs() + 1e-8), rtol=1e-6, atol=1e-6), k
    assert (net(x) * weight).sum() < loss                       # and goes down the slope


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_trainer_trains_it(tmp_path, dtype):
    torch.manual_seed(2)
    B, H, W = 4, 16, 16
    data = [(torch.rand(6, H, W), torch.rand(3, H, W)) for _ in range(2 * B)]
    cfg = TrainingConfig(batch_size=B, learning_rate=1e-3, epochs=1, device="cuda", npz_dir=tmp_path, normalize=False, base_channels=8, depth=2,
                         checkpoint_dir=tmp_path / "ck", rollout_step=1, use_early_stopping=True,
                         physics_loss=PhysicsLossConfig(enable_divergence=True, enable_gradient=True, enable_emitter=True, grid_spacing=2.0 / W))
    net = PixelNet(dtype).cuda()
    loader = DataLoader(data, batch_size=B)
    with pytest.raises(ValueError, match="autograd"):
        Trainer(net, loader, loader, cfg, "cuda")
    tr = Trainer(net, loader, loader, cfg, "cuda", engine="autograd")
    assert isinstance(tr.optimizer, ClipAdam)
    before = [p.detach().clone() for p in net.parameters()]
    tr.train()                                                   # an epoch, validation, early stopping's checkpoint and its return
    assert tr.optimizer.step_count == 2 and float(tr.optimizer.grad_norm) > 0
    assert any(not torch.equal(a, b) for a, b in zip(before, net.parameters()))
    tr.save_checkpoint(0)
    again = Trainer(PixelNet(dtype).cuda(), loader, loader, cfg, "cuda", engine="autograd")
    again.load_checkpoint(next((tmp_path / "ck").rglob("checkpoint_epoch_1.pth")))
    assert all(torch.equal(a, b) for a, b in zip(again.model.parameters(), net.parameters())) and again.optimizer.step_count == 2
    for a, b in zip(tr.optimizer._w, again.optimizer._w):
        assert (a is None and b is None) or torch.equal(a, b)
    d, e = tr.train_epoch(), again.train_epoch()
    assert d == e and all(torch.equal(a, b) for a, b in zip(again.model.parameters(), net.parameters()))


def test_the_unet_keeps_its_optimizer(tmp_path):
    from fluidnet_amd.models.unet import UNet
    from fluidnet_amd.training.optim import FusedClipAdam
    cfg = TrainingConfig(batch_size=2, learning_rate=1e-3, epochs=1, device="cuda", npz_dir=tmp_path, normalize=False, base_channels=8, depth=2,
                         checkpoint_dir=tmp_path / "ck")
    net = UNet(UNetConfig(in_channels=6, base_channels=8, depth=2), precision="fp32").cuda()
    for engine in ("plan", "autograd"):
        assert isinstance(Trainer(net, [], [], cfg, "cuda", engine=engine).optimizer, FusedClipAdam)
