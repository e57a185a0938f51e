"""A small language model made of the package's operators, trained and served.

    python examples/lm_ends.py [--steps 60] [--loss softmax|familywise|entropy] [--clip 1.0]

Training: embedding rows, one residual block, the norm of the stream, and the
loss of a tied output layer without materialised logits -- softmax cross
entropy, the same with a bonus for the entropy of its rows, or the Familywise
loss on the same operands.  Padding positions carry the ignored label.  The
gradients may be clipped to a global norm on their way into the update's
float32.  Serving: the output layer in 8-bit integers, fed by the norm's 8-bit
form, one token per sequence at a time, with the log probabilities of what was
chosen and of the likeliest alternatives.

The data is synthetic: sequences that count upwards modulo a stride each, so
that the next token follows from the two before it.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-familywise-loss_b200"))

import fwloss_b200 as fw  # noqa: E402
from fwloss_b200.lm_head import fw_lm_head_loss  # noqa: E402

VOCAB, DIM, LENGTH, BATCH, IGNORED = 1009, 256, 33, 64, -100
BONUS = 0.01  # of a nat of entropy, in nats of loss


def batch(generator, rows=BATCH):
    """(tokens [rows, L], targets [rows, L]); the ends of short sequences are ignored."""
    start = torch.randint(0, VOCAB, (rows, 1), generator=generator, device="cuda")
    stride = torch.randint(1, 8, (rows, 1), generator=generator, device="cuda")
    length = torch.randint(LENGTH // 2, LENGTH + 1, (rows, 1), generator=generator, device="cuda")
    at = torch.arange(LENGTH + 1, device="cuda")
    tokens = (start + stride * at) % VOCAB
    targets = torch.where(at[1:] < length, tokens[:, 1:], IGNORED)
    return tokens[:, :-1].contiguous(), targets


class Model:
    """Parameters in bfloat16, with the fp32 state that the updates are made in."""

    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(shape, generator=g, device="cuda") * scale

        self.master = {"embed": normal(VOCAB, DIM, scale=DIM ** -0.5), "mix": normal(2 * DIM, 4 * DIM, scale=0.05),
                       "out": normal(4 * DIM, DIM, scale=0.03), "gain1": torch.ones(DIM, device="cuda"),
                       "gain2": torch.ones(DIM, device="cuda")}
        self.grads = {k: torch.zeros_like(v) for k, v in self.master.items()}
        self.norm = None  # of the last step's gradients, where they were clipped
        self.moment = {k: (torch.zeros_like(v), torch.zeros_like(v)) for k, v in self.master.items()}
        self.step_count = 0
        self.refresh()

    def refresh(self):
        self.p = {k: v.bfloat16().requires_grad_(True) for k, v in self.master.items()}

    def stream(self, tokens):
        """(block output, stream), both [..., L, D], whose sum the last norm takes."""
        p = self.p
        x = fw.embed_tokens(tokens, p["embed"], scale=DIM ** 0.5)
        h = fw.rms_norm(x, p["gain1"])
        before = torch.nn.functional.pad(h, (0, 0, 1, 0))[..., :-1, :]  # the position before
        return torch.nn.functional.gelu(torch.cat([h, before], -1) @ p["mix"]) @ p["out"], x

    def loss(self, tokens, targets, kind):
        block, x = self.stream(tokens)
        y, _ = fw.rms_norm(block, self.p["gain2"], residual=x)
        hidden, targets = y.reshape(-1, DIM), targets.reshape(-1)
        if kind == "softmax":
            return fw.lm_head_cross_entropy(hidden, self.p["embed"], targets, ignore_index=IGNORED)
        if kind == "entropy":
            logp, entropy = fw.lm_head_log_probs(hidden, self.p["embed"], targets, ignore_index=IGNORED)
            return -(logp + BONUS * entropy).sum() / (targets != IGNORED).sum()  # both are 0 in ignored rows
        live = targets != IGNORED
        return fw_lm_head_loss(hidden[live], self.p["embed"], targets[live])

    def update(self, rate=2e-3, clip=None):
        self.step_count += 1
        if clip is not None:
            self.norm = fw.clip_grad_norm_([self.p[k].grad for k in self.p], clip, out=[self.grads[k] for k in self.p])
        for k, w in self.master.items():
            g = self.p[k].grad.float() if clip is None else self.grads[k]
            m, v = self.moment[k]
            m.lerp_(g, 0.1)
            v.lerp_(g * g, 0.02)
            w -= rate * (m / (1 - 0.9 ** self.step_count)) / ((v / (1 - 0.98 ** self.step_count)).sqrt() + 1e-8)
        self.refresh()


def train(steps=60, kind="softmax", seed=0, clip=None):
    """The trained model and the loss of every step."""
    model, g, losses = Model(seed), torch.Generator(device="cuda").manual_seed(seed + 1), []
    for _ in range(steps):
        loss = model.loss(*batch(g), kind)
        loss.backward()
        model.update(clip=clip)
        losses.append(loss.detach())
    return model, [float(x) for x in losses]


class Server:
    """Next tokens from the output layer in 8-bit integers."""

    def __init__(self, model):
        self.model = model
        self.weight, self.weight_scale = fw.quantize_rows_int8(model.p["embed"].detach())

    @torch.no_grad()
    def logits(self, tokens):
        """float32 logits [rows, V] for the position behind tokens [rows, L]."""
        block, x = self.model.stream(tokens[:, -2:])
        q, scale, _ = fw.rms_norm_int8(block[:, -1], self.model.p["gain2"], residual=x[:, -1])
        return fw.int8_linear(q, scale, self.weight, self.weight_scale, out_dtype=torch.float32)

    def generate(self, tokens, count):
        for _ in range(count):
            tokens = torch.cat([tokens, self.logits(tokens).argmax(1, keepdim=True)], 1)
        return tokens

    def score(self, tokens, following, top_k=3):
        """(log probability of the tokens [rows] that follow, entropy, log probabilities and ids of the likeliest)"""
        return fw.token_log_probs(self.logits(tokens), following, top_k=top_k)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--loss", choices=("softmax", "familywise", "entropy"), default="softmax")
    ap.add_argument("--clip", type=float, default=None, help="global norm that the gradients are clipped to")
    a = ap.parse_args()
    model, losses = train(a.steps, a.loss, clip=a.clip)
    for i in range(0, a.steps, max(1, a.steps // 8)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"last       loss {losses[-1]:.4f}")
    tokens, _ = batch(torch.Generator(device="cuda").manual_seed(99), 4)
    print("prompts and their continuation, 8-bit output layer:")
    server = Server(model)
    for row in server.generate(tokens[:, :4], 6).tolist():
        print("  ", row[:4], "->", row[4:])
    logp, entropy, top_logp, top_ids = server.score(tokens[:, :4], tokens[:, 4])
    print("the tokens that followed, and the likeliest:")
    for i in range(4):
        likeliest = ", ".join(f"{t} {v:.3f}" for t, v in zip(top_ids[i].tolist(), top_logp[i].tolist()))
        print(f"   {int(tokens[i, 4])} {float(logp[i]):.3f} (entropy {float(entropy[i]):.3f}): {likeliest}")


if __name__ == "__main__":
    main()
