"""Training with the RepUNet's norms and with 32- or 8-bit optimizer state, through step_batch on one GPU.

  step    time of a training step and peak memory, RepUNet [3, 5], 8 x 1 x 512 x 512 bf16
  losses  800 steps on synthetic discs (4 x 1 x 64 x 64, features 16, 32), mean loss of the last 50, three seeds
"""
import logging
import os
import sys
import time
import types

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from unet_amd.models import REGISTRY                            # noqa: E402
from unet_amd.utils.builders import build_loss, get_optim       # noqa: E402
from unet_amd.utils.train_step import step_batch                # noqa: E402

DEV = torch.device("cuda:0")


def trainer(kind, norm, bits, features, lr):
    kw = {"features": list(features)}
    if kind == "reparam_unet":
        kw.update(kernel_sizes=[3, 5], norm=norm)
    model = REGISTRY[kind](in_channels=1, n_classes=2, **kw).to(DEV).train()
    opt = get_optim("adamw", model.parameters(), lr=lr, weight_decay=1e-4, **({"state_bits": 8} if bits == 8 else {}))
    loss = build_loss("ce_dice", dict(ce_weight=1.0, dice_weight=1.0, ignore_index=255), DEV)
    return types.SimpleNamespace(optimizer=opt, amp=True, model=model, grad_clip=1.0, cbs=[], current_epoch=1, loss_fn=loss,
                                 logger=logging.getLogger("bench"))


def steps(norm, bits, n=20):
    torch.manual_seed(0)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    t = trainer("reparam_unet", norm, bits, (64, 128, 256, 512), 1e-4)
    scaler = torch.amp.GradScaler("cuda", enabled=False)
    x = torch.rand(8, 1, 512, 512, device=DEV)
    y = (x[:, 0] > 0.7).long()
    for k in range(5):
        step_batch(t, x, y, scaler, k)
    best = 1e9
    for _ in range(3):
        torch.cuda.synchronize()
        a = time.perf_counter()
        for k in range(n):
            step_batch(t, x, y, scaler, k)
        torch.cuda.synchronize()
        best = min(best, (time.perf_counter() - a) / n)
    print(f"step: RepUNet [3, 5] {norm} norm, {bits}-bit state: {best * 1e3:.2f} ms, peak {torch.cuda.max_memory_allocated() / 2 ** 30:.2f} GiB", flush=True)


def discs(g, n=4, s=64):
    yy, xx = torch.meshgrid(torch.arange(s), torch.arange(s), indexing="ij")
    c, r = torch.rand((n, 2, 1, 1), generator=g) * s, torch.rand((n, 1, 1), generator=g) * s / 4 + 4
    y = ((yy - c[:, 0]) ** 2 + (xx - c[:, 1]) ** 2 < r ** 2).long()
    return (y[:, None] * 0.5 + 0.4 * torch.randn((n, 1, s, s), generator=g)), y


def losses(kind, norm, bits, count=800):
    out = []
    for seed in (1, 2, 3):
        torch.manual_seed(seed)
        g = torch.Generator().manual_seed(seed)
        t = trainer(kind, norm, bits, (16, 32), 1e-3)
        scaler = torch.amp.GradScaler("cuda", enabled=False)
        last = []
        for k in range(count):
            x, y = discs(g)
            loss = step_batch(t, x.to(DEV), y.to(DEV), scaler, k)[2]["main_loss"]
            last = (last + [loss])[-50:]
        out.append(sum(last) / len(last))
    name = "U-Net" if kind == "unet" else f"RepUNet [3, 5] {norm} norm"
    print(f"losses: {name} (16, 32), {bits}-bit state: " + " / ".join(f"{v:.4f}" for v in out), flush=True)


if __name__ == "__main__":
    for norm, bits in (("group", 32), ("group", 8), ("layer", 32), ("layer", 8)):
        steps(norm, bits)
    for kind, norm in (("unet", None), ("reparam_unet", "layer"), ("reparam_unet", "group")):
        for bits in (32, 8):
            losses(kind, norm, bits)
