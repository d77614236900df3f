"""How far the LoRA towers' adapter gradients lie from the native ones when what their backward reads is kept in 8 bits
(`lora_checkpoint: int8`): relative distance and cosine per tower and the farthest single adapter, per recompute policy, at
siglip_sequential's full size (SigLIP base, 384 pixels, T = 4, fp16; random weights and data).
    python tools/lora_checkpoint_error.py [batch] [outlier]   (outlier: added to one column of the position embeddings)"""
import os
import sys
import warnings

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bench  # noqa: E402
from bifold.losses import Losses  # noqa: E402
from bifold.models import Models  # noqa: E402

dev = torch.device("cuda:0")
batch = int(sys.argv[1]) if len(sys.argv) > 1 else 8
outlier = float(sys.argv[2]) if len(sys.argv) > 2 else 0.0
sample = bench.synthetic_sequential_batch(batch, dev, seed=3407)
loss_fn = Losses.get_by_name(cfg=dict(name="bce_gaussmap", is_bimanual=True, mask_pick_heatmap=False))


def gradients(policy, how):
    torch.manual_seed(3407)
    cfg = dict(name="siglip_sequential", image_size=384, is_bimanual=True, requires_graph=False, patch_size=16,
               automodel_name="google/siglip-base-patch16-384", dim=768, emb_dropout=0.0, lora=True, r=8, lora_alpha=32,
               lora_dropout=0.0, target_modules=["q_proj", "v_proj"], threshold=0.5, text_encoder=None,
               pick_place_model="pick_place_convdecoder", fusion_model="concat_transformer", depth=8, heads=16,
               mlp_ratio=4, dropout=0.0, dtype="fp16", context_length=4, lora_recompute=policy, lora_checkpoint=how)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        model = Models.get_by_name(cfg, device=dev)
    with torch.no_grad():
        g = torch.Generator().manual_seed(6)
        for n, p in model.named_parameters():
            if ".lora_B." in n:
                p.copy_(torch.randn(p.shape, generator=g) * 0.02)
            if n.endswith("position_embedding.weight"):
                p[:, 5] += outlier
    model = model.to(dev).train()
    loss, _ = loss_fn(model(sample), sample)
    model.zero_grad()
    loss.backward()
    torch.cuda.synchronize()
    return {n: p.grad.detach().double().flatten() for n, p in model.named_parameters() if p.requires_grad and ".lora_" in n}


def far(a, b):
    return ((a - b).norm() / b.norm()).item()


native = gradients("none", "native")                            # the same bits under every policy
for policy in ("none", "mlp", "full"):
    got = gradients(policy, "int8")
    for tower in ("vision_model", "text_model"):
        names = [n for n in native if tower in n]
        a, b = torch.cat([got[n] for n in names]), torch.cat([native[n] for n in names])
        worst = max(names, key=lambda n: far(got[n], native[n]))
        cos = (torch.dot(a, b) / (a.norm() * b.norm())).item()
        print(f"B={batch} outlier={outlier:g} lora_recompute={policy:4s} {tower:12s} relative distance {far(a, b):.4f}, cosine "
              f"{cos:.6f}, farthest adapter {far(got[worst], native[worst]):.4f} ({worst.split('encoder.')[-1]})", flush=True)
