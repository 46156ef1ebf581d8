"""A recurrent logic-gate network over tokens: trained from 8-bit checkpoints, decoded by beam search.

    python examples/token_logic_net.py [--steps 300] [--beams 4]

The soft network reads a token through a scaled embedding (squashed to [0, 1]), joins it with
its recurrent state in a layer of logic gates, and reads one group of gates per vocabulary
token as that token's logit.  Training unrolls it over the sequence; inside ``checkpoint8()`` every
unrolled layer keeps its input in 8 bits.  Decoding runs the hard circuit: the embedding's signs
and the state are bit-packed samples (one per beam), and after each ``beam_step`` the packed state
is reordered by the chosen beams.

The task is synthetic: sequences that count on in steps of 1, 2 or 3 modulo the vocabulary.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import silogic_b200 as silogic                                   # noqa: E402
from silogic_b200.bitpacking import convert_layer, pack_bits, unpack_bits   # noqa: E402


class TokenLogicNet(nn.Module):
    def __init__(self, vocab, dim=64, state=256, per_token=16, k=8, tau=2.0, seed=0):
        super().__init__()
        self.vocab, self.state_dim = vocab, state
        self.embed = silogic.TokenEmbedding(vocab, dim)
        self.cell = silogic.LogicLayer(dim + state, state, node="walsh", k=k, seed=seed)
        self.read = silogic.LogicLayer(state, vocab * per_token, node="walsh", k=k, seed=seed + 1)
        self.head = silogic.GroupSum(vocab, tau=tau)

    def forward(self, ids):
        """[B, T] tokens -> [B, T, vocab] logits of the next token (soft, differentiable)."""
        h = torch.full((ids.shape[0], self.state_dim), 0.5, device=ids.device)
        out = []
        for x in torch.sigmoid(self.embed(ids)).unbind(1):
            h = self.cell(torch.cat([x, h], 1))
            out.append(self.head(self.read(h)))
        return torch.stack(out, 1)

    @torch.no_grad()
    def circuit(self):
        """The hard step: (token ids [n], packed state) -> (logits [n, vocab], packed state)."""
        cell, read = convert_layer(self.cell), convert_layer(self.read)

        def step(ids, h):
            x = pack_bits((silogic.token_embedding(ids, self.embed.weight) > 0).to(torch.uint8))
            h = cell(torch.cat([x, h[:, :x.shape[1]]], 0))       # 64 beams to a word
            counts = self.head.forward_hard(unpack_bits(read(h), ids.numel()))
            return counts / self.head.tau, h
        return step

    @torch.no_grad()
    def generate(self, prompt, steps, beams=4):
        """Beam search from ``prompt`` [B, T]; returns ([B, beams, steps] tokens, [B, beams] scores)."""
        B, dev = prompt.shape[0], prompt.device
        step = self.circuit()
        h = pack_bits(torch.zeros((B, self.state_dim), dtype=torch.uint8, device=dev))
        for t in range(prompt.shape[1]):
            logits, h = step(prompt[:, t].contiguous(), h)
        # one beam per entry becomes `beams`
        r = silogic.beam_step(logits, torch.zeros((B, 1), device=dev), width=beams)
        h = silogic.beam_reorder(h, r.parents, layout="packed", beams=1)
        tokens = r.tokens.unsqueeze(2)
        for _ in range(steps - 1):
            logits, h = step(r.tokens.reshape(-1), h)
            r = silogic.beam_step(logits, r.scores)
            h = silogic.beam_reorder(h, r.parents, layout="packed")
            tokens = silogic.beam_reorder(tokens.reshape(B * beams, -1), r.parents).view(B, beams, -1)
            tokens = torch.cat([tokens, r.tokens.unsqueeze(2)], 2)
        return tokens, r.scores


def batch(n, length, vocab, gen, device):
    start = torch.randint(0, vocab, (n, 1), generator=gen)
    stride = torch.randint(1, 4, (n, 1), generator=gen)
    return ((start + stride * torch.arange(length)) % vocab).to(device)


def train(net, steps, batch_size=256, length=8, lr=0.03, device="cuda", log=print):
    gen = torch.Generator().manual_seed(0)
    opt = torch.optim.Adam(net.parameters(), lr=lr)
    for i in range(steps):
        ids = batch(batch_size, length + 1, net.vocab, gen, device)
        with silogic.checkpoint8():
            logits = net(ids[:, :-1])
        loss = F.cross_entropy(logits[:, 1:].flatten(0, 1), ids[:, 2:].flatten())   # one token tells no stride
        opt.zero_grad()
        loss.backward()
        opt.step()
        if log and (i % 50 == 0 or i == steps - 1):
            log(f"step {i:4d}  loss {loss.item():.3f}")
    return loss.item()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--vocab", type=int, default=24)
    ap.add_argument("--beams", type=int, default=4)
    a = ap.parse_args()
    torch.manual_seed(0)
    net = TokenLogicNet(a.vocab).cuda()
    train(net, a.steps)
    prompt = batch(4, 4, a.vocab, torch.Generator().manual_seed(1), "cuda")
    tokens, scores = net.generate(prompt, 6, a.beams)
    for p, t, s in zip(prompt.tolist(), tokens.tolist(), scores.tolist()):
        print(p, "->", t[0], f"({s[0]:.2f})")


if __name__ == "__main__":
    main()
