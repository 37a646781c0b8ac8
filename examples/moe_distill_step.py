"""Quantization-aware training of a small mixture-of-experts model by distillation.

A teacher with full-precision experts writes down its top logits once.  A
student of the same architecture, its experts quantized by the soft trellis
quantizer at a falling temperature, is trained to give the same distribution:

    moe_route               which expert each token goes to
    bcjr_quantize_experts   every expert's quantized weights in one call
    grouped_matmul          the experts' products over ragged groups of tokens
    moe_combine             each token's weighted sum
    topk_distill_loss       divergence from the teacher's top logits

and the gradient runs back through all of them into the latent weights.

    python examples/moe_distill_step.py [--steps 30]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quant-2bit_amd"))
import bcjr  # noqa: E402

VOCAB, HIDDEN, INTER, EXPERTS, TOP_K = 2000, 128, 64, 8, 2
L, K_BITS, V_DIM = 12, 2, 1  # 2 bits a weight, 4,096 states


class Model:
    """Embedding, one mixture-of-experts layer, head.  The latent weights of the
    experts are what is trained."""

    def __init__(self, seed, device):
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, device=device, generator=g) * scale

        self.embed = normal(VOCAB, HIDDEN).bfloat16()
        self.router = normal(EXPERTS, HIDDEN, scale=HIDDEN ** -0.5).bfloat16()
        self.gate_up = [normal(2 * INTER, HIDDEN, scale=HIDDEN ** -0.5) for _ in range(EXPERTS)]
        self.down = [normal(HIDDEN, INTER, scale=INTER ** -0.5) for _ in range(EXPERTS)]
        self.head = normal(VOCAB, HIDDEN, scale=3 * HIDDEN ** -0.5).bfloat16()
        self.codebook = bcjr.make_1mad_codebook(L, device)
        self.signs = [tuple(torch.as_tensor(bcjr.make_sign_vector(n, 7 * i + j), device=device)
                            for j, n in enumerate(w.shape)) for i, w in enumerate(self.gate_up + self.down)]

    def experts(self, temperature=None):
        """(gate_up (E, 2I, H), down (E, H, I)), quantized at a temperature."""
        latent = self.gate_up + self.down
        if temperature is not None:
            latent = bcjr.bcjr_quantize_experts(latent, [s[0] for s in self.signs], [s[1] for s in self.signs],
                                                self.codebook, temperature, L=L, k=K_BITS, V=V_DIM)
        return torch.stack(latent[:EXPERTS]), torch.stack(latent[EXPERTS:])

    def logits(self, tokens, experts, valid=None):
        """(T, VOCAB) of T tokens; padding (valid False) passes the experts by."""
        gate_up, down = experts
        x = F.embedding(tokens, self.embed)
        route = bcjr.moe_route(x @ self.router.t(), TOP_K, renormalize=True, valid=valid)
        h = bcjr.grouped_matmul(x, gate_up, route.offsets, rows=route.rows, slots=route.slots)
        gate, up = h.chunk(2, dim=1)
        y = bcjr.grouped_matmul(F.silu(gate) * up, down, route.offsets)
        return (x + bcjr.moe_combine(y, route.weights, route.rows, route.slots)) @ self.head.t()


def main(steps=30, tokens=512, top=32, temperature=2.0, device="cuda:0", verbose=True):
    """Train for some steps; returns the loss of each."""
    model = Model(0, torch.device(device))
    g = torch.Generator(device=device)
    g.manual_seed(1)
    batch = torch.randint(0, VOCAB, (tokens,), device=device, generator=g)
    valid = torch.arange(tokens, device=device) < tokens - tokens // 16  # the batch ends in padding
    weight = valid.float() / valid.sum()

    with torch.no_grad():  # the teacher: its top logits and their normaliser are kept
        teacher = model.logits(batch, model.experts(), valid).float()
        values, indices = torch.topk(teacher, top, dim=1)
        lse = torch.logsumexp(teacher / temperature, dim=1)

    latent = model.gate_up + model.down
    for w in latent:
        w.requires_grad_()
    opt = torch.optim.Adam(latent, lr=2e-3)
    losses = []
    for step in range(steps):
        T = bcjr.cosine_temperature_schedule(step, steps, 0.3, 0.1)
        opt.zero_grad(set_to_none=True)
        logits = model.logits(batch, model.experts(T), valid)
        # the rows' weights are known, so loss and gradient come from one launch ...
        loss, g_logits = bcjr.topk_distill_loss_and_grad(logits, values, indices, weight, temperature=temperature,
                                                         teacher_lse=lse)
        logits.backward(g_logits)
        opt.step()
        losses.append(float(loss @ weight))
        if verbose and step % 5 == 0:
            print(f"step {step:3d}  T {T:.3f}  loss {losses[-1]:.5f}", flush=True)
    # ... and the same loss through autograd, for a loss that joins others
    logits = model.logits(batch, model.experts(0.1), valid)
    final = (bcjr.topk_distill_loss(logits, values, indices, temperature=temperature, teacher_lse=lse) * weight).sum()
    final.backward()
    losses.append(float(final.detach()))
    if verbose:
        print(f"trained: loss {losses[-1]:.5f}", flush=True)
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    main(ap.parse_args().steps)
