"""Serves a batch of prompts of different lengths from a paged KV cache.

Every step feeds some sequences a piece of their prompt while others, whose
prompts are done, decode one token: new K/V rows are appended to the pages, the
ragged chunk attends over them, every key's attention weight is collected, and
sequences that outgrow the budget keep their most attended keys.

    python examples/serve_paged.py --normalizer entmax15 --budget 256 --recent 32

The model is a randomly initialised Qwen3 (no weights are downloaded).
"""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from transformers import Qwen3Config, Qwen3ForCausalLM  # noqa: E402
from transformers.models.qwen3.modeling_qwen3 import apply_rotary_pos_emb  # noqa: E402

from hf_attention_normalizers_b200.serving import PagedServingCache  # noqa: E402


def small_model(device="cuda", dtype=torch.bfloat16, layers=4):
    config = Qwen3Config(vocab_size=1024, hidden_size=512, intermediate_size=1024, num_hidden_layers=layers,
                         num_attention_heads=8, num_key_value_heads=2, head_dim=64, max_position_embeddings=8192)
    torch.manual_seed(0)
    return Qwen3ForCausalLM(config).to(device=device, dtype=dtype).eval()


def forward_step(model, cache, step, tokens, positions, normalizer):
    """Logits [T, vocab] of the packed new tokens; ``positions`` are their places in the text."""
    hidden = model.model.embed_tokens(tokens)
    cos, sin = model.model.rotary_emb(hidden[None], positions[None])
    for index, layer in enumerate(model.model.layers):
        attn, x = layer.self_attn, layer.input_layernorm(hidden)
        shape = (x.shape[0], -1, attn.head_dim)
        q, k = attn.q_norm(attn.q_proj(x).view(shape)), attn.k_norm(attn.k_proj(x).view(shape))
        q, k = apply_rotary_pos_emb(q[None], k[None], cos, sin, unsqueeze_dim=2)
        cache.append(index, step, k[0].contiguous(), attn.v_proj(x).view(shape))
        out = cache.attend(index, step, q[0].contiguous(), normalizer)
        hidden = hidden + attn.o_proj(out.reshape(x.shape[0], -1))
        hidden = hidden + layer.mlp(layer.post_attention_layernorm(hidden))
    return model.lm_head(model.model.norm(hidden))


@torch.no_grad()
def generate(model, prompts, new_tokens, normalizer="softmax1", piece=128, budget=None, recent=32, block_size=32):
    """Greedy continuation of every prompt (lists of token ids); returns the generated ids."""
    device = model.lm_head.weight.device
    total = max(len(p) for p in prompts) + new_tokens
    longest = min(total, budget + piece) if budget is not None else total
    config = model.config
    cache = PagedServingCache(config.num_hidden_layers, len(prompts), len(prompts) * -(-longest // block_size), block_size,
                              config.num_key_value_heads, config.head_dim, model.lm_head.weight.dtype, device,
                              track_weights=budget is not None)
    seen = [0] * len(prompts)
    out = [[] for _ in prompts]
    while any(len(o) < new_tokens for o in out):
        chunk, counts = [], []
        for p, s, o in zip(prompts, seen, out):
            rest = p[s:s + piece] if s < len(p) else (o[-1:] if len(o) < new_tokens else [])
            chunk.append(rest)
            counts.append(len(rest))
        step = cache.step(counts)
        tokens = torch.tensor([t for c in chunk for t in c], device=device)
        positions = torch.tensor([s + i for s, n in zip(seen, counts) for i in range(n)], device=device)
        logits = forward_step(model, cache, step, tokens, positions, normalizer)
        last = torch.tensor(counts).cumsum(0) - 1
        best = logits[last.clamp_min(0)].argmax(-1).tolist()
        for b, n in enumerate(counts):
            seen[b] += n
            if n and seen[b] >= len(prompts[b]):
                out[b].append(best[b])
        if budget is not None:
            cache.evict(budget, recent)
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--normalizer", default="softmax1", choices=["softmax1", "sparsemax", "entmax15"])
    ap.add_argument("--budget", type=int, default=None)
    ap.add_argument("--recent", type=int, default=32)
    ap.add_argument("--new-tokens", type=int, default=32)
    a = ap.parse_args()
    model = small_model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (700, 33, 260, 1)]
    generate(model, prompts, 2, a.normalizer, budget=a.budget, recent=a.recent)  # warm-up
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = generate(model, prompts, a.new_tokens, a.normalizer, budget=a.budget, recent=a.recent)
    dt = time.perf_counter() - t
    for p, o in zip(prompts, out):
        print(f"prompt of {len(p):4d}: {o[:8]} ...")
    done = sum(len(p) for p in prompts) + sum(len(o) for o in out)
    print(f"{done} tokens in {dt:.3f} s ({done / dt:.0f} tokens/s)")


if __name__ == "__main__":
    main()
