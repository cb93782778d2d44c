"""Distil a small language model from a teacher's top logits.

    python examples/distill.py [--steps 20] [--top_k 16] [--temperature 2.0]

The teacher scores each batch once and keeps its top-K logits per token. The student (tied, scaled embeddings; a
head loss without materialised logits) trains on the divergence from them mixed with the cross-entropy of the next
token. Seeded synthetic tokens; bf16 on CUDA, fp32 on the CPU.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from nano_train_b200.config import FullPrecisionResolver, ModelConfig  # noqa: E402
from nano_train_b200.models.transformer import TransformerModel  # noqa: E402
from nano_train_b200.parallel.flat_optimizer import FlatAdamW, split_decay_groups  # noqa: E402


def build(hidden: int, layers: int, vocab: int, device: torch.device, dtype: torch.dtype, **kw) -> TransformerModel:
    return TransformerModel(ModelConfig(
        param_dtype=dtype, param_device=device, precision_resolver=FullPrecisionResolver(), hidden_size=hidden,
        num_layers=layers, num_attention_heads=max(1, hidden // 64), intermediate_size=2 * hidden, vocab_size=vocab,
        max_position_embeddings=512, dropout=0.0, norm="rmsnorm", position="rope", mlp="swiglu", bias=False, **kw))


@torch.no_grad()
def top_logits(teacher: TransformerModel, ids: torch.Tensor, k: int):
    """The teacher's k largest logits of every position, as a store of them would hold them."""
    values, indices = teacher(ids).float().topk(k, dim=-1)
    return values, indices


def main():
    ap = argparse.ArgumentParser(description="distillation from top logits")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch_size", type=int, default=4)
    ap.add_argument("--seq_len", type=int, default=64)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--hidden_size", type=int, default=128)
    ap.add_argument("--top_k", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=2.0)
    ap.add_argument("--label_weight", type=float, default=0.25)
    ap.add_argument("--lr", type=float, default=2e-3)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    dtype = torch.bfloat16 if dev.type == "cuda" else torch.float32
    torch.manual_seed(a.seed)
    teacher = build(2 * a.hidden_size, 2, a.vocab, dev, dtype, tie_word_embeddings=False, init_std=0.1).eval()
    student = build(a.hidden_size, 2, a.vocab, dev, dtype, tie_word_embeddings=True, fused_head_loss=True,
                    embedding_scale=math.sqrt(a.hidden_size))
    optimizer = FlatAdamW(split_decay_groups(student, 0.01), lr=a.lr, max_grad_norm=1.0)
    g = torch.Generator().manual_seed(a.seed)
    batches = []
    for _ in range(4):  # a few batches, seen again and again
        ids = torch.randint(0, a.vocab, (a.batch_size, a.seq_len + 1), generator=g).to(dev)
        batches.append((ids[:, :-1], ids[:, 1:], *top_logits(teacher, ids[:, :-1], a.top_k)))
    for step in range(a.steps):
        ids, labels, values, indices = batches[step % len(batches)]
        optimizer.zero_grad()
        loss = student.forward_distill_loss(ids, values, indices, labels, temperature=a.temperature,
                                            label_weight=a.label_weight)
        loss.backward()
        optimizer.step()
        if step % 5 == 0 or step == a.steps - 1:
            with torch.no_grad():
                hard = student.forward_loss(ids, labels)
            print(f"step {step} loss {float(loss.detach()):.4f} cross-entropy {float(hard):.4f}")


if __name__ == "__main__":
    main()
