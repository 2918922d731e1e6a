"""Serving of ragged requests on a paged 4-bit KV cache with drafted tokens.

``PagedLlama`` is the quantized Llama of ``QuantizedModel`` written over
``Backend``'s ops, for requests that come and go: each has its own length,
pages of the cache are handed out on the GPU (``KV4Plan``), rows are appended
in 4 bits (``KV4AppendRoPE``), attention reads them through the block table
(``KV4Attention``), and drafted tokens are checked together (``VerifyDraft``).

    python -m tendo_b200.paged            # a few prompts through a small model

Drafts come from prompt lookup: what followed the last token where it stood
before.  They cost no model, and are certain as a drafter's distribution goes,
so ``VerifyDraft`` takes no draft probabilities.
"""
from __future__ import annotations

from . import (MATS_PER_LAYER, STREAM_EMBED, STREAM_LMHEAD, Backend, ShapeError, synth_tokens)

MAT_Q, MAT_K, MAT_V, MAT_O, MAT_GATE, MAT_UP, MAT_DOWN = range(7)


class PagedLlama:
    """Quantized Llama with synthetic weights (the engine's draws) over a pool of 4-bit cache pages."""

    def __init__(self, cfg: dict, num_blocks: int, block_size: int = 16, max_requests: int = 64, seed: int = 0,
                 device: int = 0):
        import torch

        self.cfg, self.block, self.be = dict(cfg), block_size, Backend(device)
        be, dev = self.be, f"cuda:{device}"
        d, H, Hkv, F, V = (cfg[k] for k in ("dim", "heads", "kv_heads", "hidden", "vocab"))
        self.D = d // H
        self.layers = []
        for layer in range(cfg["layers"]):
            def mat(m, n, k):
                return be.SynthQuantized(n, k, seed, layer * MATS_PER_LAYER + m)

            def join(*parts):  # rows of several Linears as one, so that one product makes them all
                return tuple(torch.cat(p).contiguous() for p in zip(*parts))

            self.layers.append(dict(
                qkv=join(mat(MAT_Q, H * self.D, d), mat(MAT_K, Hkv * self.D, d), mat(MAT_V, Hkv * self.D, d)),
                o=mat(MAT_O, d, H * self.D), gate=mat(MAT_GATE, F, d), up=mat(MAT_UP, F, d), down=mat(MAT_DOWN, d, F),
                pages=be.KV4Pages(num_blocks, Hkv, self.D, block_size)))
        self.norm = torch.ones(d, device=dev)
        self.embed = be.SynthNormal(V, d, seed, STREAM_EMBED, 0.02)
        self.lm_head = be.SynthNormal(V, d, seed, STREAM_LMHEAD, 0.02)
        self.cos, self.sin = (torch.from_numpy(t).to(dev) for t in be.RoPETables(self.D, cfg["max_seq"],
                                                                                 cfg["rope_base"]))
        columns = -(-cfg["max_seq"] // block_size)
        self.table = torch.full((max_requests, columns), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.count = torch.tensor([num_blocks], dtype=torch.int32, device=dev)
        self.held = [0] * max_requests  # positions that each request has pages for
        self.dev = dev

    def _plan(self, ctx, new):
        """Plans ctx kept and new added positions per request; a plan that does not fit raises and changes nothing."""
        import torch

        # the block table's last page may reach further than the RoPE tables do
        most = max(c + n for c, n in zip(ctx, new))
        if most > self.cfg["max_seq"]:
            raise ShapeError(f"a request of {most} positions, the model takes {self.cfg['max_seq']}")
        lens = torch.tensor([self.held, ctx, new], dtype=torch.int32, device=self.dev)
        step = self.be.KV4Plan(lens[0], lens[1], lens[2], self.table, self.free, self.count, sum(new), self.block)
        if int(step.bad):
            raise ShapeError(f"the cache has no room for {sum(new)} more positions")
        self.count = step.free_count
        self.held = [c + n for c, n in zip(ctx, new)]
        return step

    def forward(self, tokens, ctx, new):
        """Logits [T, V] of every row: request b keeps ctx[b] cached positions and adds new[b] of `tokens` [T]."""
        be, cfg = self.be, self.cfg
        H, Hkv, D, eps = cfg["heads"], cfg["kv_heads"], self.D, cfg["eps"]
        step = self._plan(ctx, new)
        x = be.Embedding(self.embed, tokens)
        T = x.shape[0]
        for w in self.layers:
            h = be.RMSNorm(x, (cfg["dim"],), self.norm, eps)
            rows = be.DequantizeMatmul(h, *w["qkv"]).view(T, H + 2 * Hkv, D)
            q = be.KV4AppendRoPE(w["pages"], rows[:, H:H + Hkv], rows[:, H + Hkv:], self.cos, self.sin, step.positions,
                                 step.slots, q=rows[:, :H])
            a = be.KV4Attention(q, w["pages"], self.table, step.seq_lens, step.q_start, max(new))
            x, h = be.AddRMSNorm(be.DequantizeMatmul(a.view(T, H * D), *w["o"]), x, self.norm, eps)
            act = be.SiLUMul(be.DequantizeMatmul(h, *w["gate"]), be.DequantizeMatmul(h, *w["up"]))
            x = be.Add(be.DequantizeMatmul(act, *w["down"]), x)
        return be.MatMulNT(be.RMSNorm(x, (cfg["dim"],), self.norm, eps), self.lm_head)

    @staticmethod
    def lookup(seq, most: int):
        """Up to `most` tokens that followed the last token of `seq` where it stood before."""
        for i in range(len(seq) - 2, -1, -1):
            if seq[i] == seq[-1]:
                return seq[i + 1:i + 1 + most]
        return []

    def generate(self, prompts, n_new: int, drafts: int = 4, temperature: float = 1.0, seed: int = 0):
        """n_new sampled tokens for each prompt (lists of ints), all in one batch; returns (sequences' new tokens,
        target passes).  Pages go back to the pool when a request has its tokens."""
        import torch

        if len(prompts) > len(self.held):
            raise ShapeError(f"{len(prompts)} prompts, room for {len(self.held)} requests")
        if not all(len(p) for p in prompts):
            raise ShapeError("a prompt without tokens has no next token")
        if not temperature > 0:
            raise ShapeError(f"temperature {temperature}: logits are divided by it, so it has to be above 0")
        most = max((len(p) for p in prompts), default=0) + n_new - 1  # the last token's own position is not taken
        if most > self.cfg["max_seq"]:
            raise ShapeError(f"{most} positions for a prompt and its tokens, the model takes {self.cfg['max_seq']}")
        B, N, V, K = len(prompts), len(self.held), self.cfg["vocab"], drafts
        gen = torch.Generator(device=self.dev)
        gen.manual_seed(seed)
        seqs = [list(map(int, p)) for p in prompts]
        want = [len(p) + n_new for p in prompts]
        cached, passes = [0] * B, 0
        while any(len(s) < w for s, w in zip(seqs, want)):
            todo = [[] for _ in range(N)]  # rows of this pass
            proposed = [[] for _ in range(B)]
            for b in range(B):
                if len(seqs[b]) < want[b]:
                    if cached[b]:  # no drafts beside a prompt
                        proposed[b] = self.lookup(seqs[b], min(K, want[b] - len(seqs[b]) - 1))
                    todo[b] = seqs[b][cached[b]:] + proposed[b]
            new = [len(t) for t in todo]
            ctx = [cached[b] if b < B and new[b] else 0 for b in range(N)]
            flat = torch.tensor([t for rows in todo for t in rows], dtype=torch.int64, device=self.dev)
            probs = self.be.Softmax(self.forward(flat, ctx, new).div_(temperature), -1)
            passes += 1
            # row i of a request's check is the distribution after its i-th proposed token
            live = [b for b in range(B) if new[b]]
            last, ends = [], 0
            for b in live:
                ends += new[b]
                last.append(ends - 1 - len(proposed[b]))
            at = torch.tensor([[min(f + i, f + len(proposed[b])) for i in range(K + 1)] for f, b in zip(last, live)],
                              device=self.dev)
            x = torch.tensor([(proposed[b] + [0] * K)[:K] for b in live], dtype=torch.int64, device=self.dev)
            lens = torch.tensor([len(proposed[b]) for b in live], dtype=torch.int32, device=self.dev)
            u = torch.rand(len(live), K + 1, generator=gen, device=self.dev)
            tokens, accepted = self.be.VerifyDraft(probs[at], x.view(len(live), K), u, draft_lens=lens)
            self.be.KV4Check()
            for b, row, n in zip(live, tokens.tolist(), accepted.tolist()):
                cached[b] = len(seqs[b]) + n  # the refused rows' positions are given up
                seqs[b] += row[:n + 1]
                if len(seqs[b]) >= want[b]:
                    cached[b] = 0
        self._plan([0] * N, [0] * N)  # every page back
        return [s[len(p):] for s, p in zip(seqs, prompts)], passes


def main():
    cfg = dict(vocab=2000, dim=512, layers=4, heads=8, kv_heads=2, hidden=1408, max_seq=512, rope_base=10000.0,
               eps=1e-5)
    model = PagedLlama(cfg, num_blocks=256, max_requests=8)
    prompts = [synth_tokens(n, cfg["vocab"], n).tolist() for n in (7, 33, 120, 64)]
    for drafts in (0, 4):
        out, passes = model.generate(prompts, 48, drafts=drafts, temperature=0.05)
        print(f"{drafts} drafts: {sum(map(len, out))} tokens in {passes} passes; first: {out[0][:8]}")
    print(f"{int(model.count)} of {model.free.numel()} pages free")


if __name__ == "__main__":
    main()
