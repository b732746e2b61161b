"""Steps over a block cache whose sequences share prefixes, and their attention in 64 bits."""
import random

import torch

BLOCK = 64


class Step:
    """``groups``: (sequences, tokens shared) pairs; ``own``: cached tokens of every sequence's own
    behind its prefix; ``news``: tokens each brings.  Blocks lie in random order; what no sequence
    holds (whole blocks, and rows behind a sequence's last token) is ``poison``."""

    def __init__(self, groups, own, news, nh, nkv, hd, dtype, seed=0, poison=float("nan"), device="cuda",
                 spread=1.0, shared_values=False):
        rng = random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        B = len(news)
        prefix = [0] * B
        for members, p in groups:
            for b in members:
                prefix[b] = p
        self.starts = [prefix[b] + own[b] for b in range(B)]
        ends = [s + n for s, n in zip(self.starts, news)]
        need = [-(-e // BLOCK) for e in ends]
        n_blocks = sum(p // BLOCK for _, p in groups) + sum(need[b] - prefix[b] // BLOCK for b in range(B)) + 2
        free = list(range(n_blocks))
        rng.shuffle(free)
        self.slots = rng.sample(range(B + 2), B)
        table = torch.full((B + 2, max(need) + 1), -1, dtype=torch.int32)
        kc = torch.full((n_blocks, nkv, BLOCK, hd), poison, dtype=torch.float32)
        vc = kc.clone()

        def fill(blk, rows):
            kc[blk, :, :rows] = spread * torch.randn((nkv, rows, hd), generator=gen)
            vc[blk, :, :rows] = torch.randn((nkv, rows, hd), generator=gen)
        for members, p in groups:
            for i in range(p // BLOCK):
                blk = free.pop()
                fill(blk, BLOCK)
                for b in members:
                    table[self.slots[b], i] = blk
        for b in range(B):
            for i in range(prefix[b] // BLOCK, need[b]):
                blk = free.pop()
                table[self.slots[b], i] = blk
                fill(blk, min(BLOCK, ends[b] - i * BLOCK))
        self.groups, self.news, self.nh, self.nkv, self.hd, self.dtype = groups, news, nh, nkv, hd, dtype
        T = sum(news)
        self.T, self.B = T, B
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        self.cu_host = cu
        self.pos_host = [self.starts[b] + i for b in range(B) for i in range(news[b])]
        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.table = table.to(device)
        self.kc = kc.to(device=device, dtype=dtype)
        self.vc = self.kc if shared_values else vc.to(device=device, dtype=dtype)
        self.tok_pos, self.cu, self.seq_slot = as_int(self.pos_host), as_int(cu), as_int(self.slots)
        # rows as a projection leaves them, with the step's keys and values behind the queries
        self.rows = torch.randn((T + 3, (nh + 2 * nkv) * hd), generator=gen).to(device=device, dtype=dtype)
        self.q = self.rows[:T, :nh * hd]
        self.scale = hd ** -0.5

    def plan(self, ops, starts=None):
        return ops.shared_prefix_plan(self.groups, self.news, starts or self.starts, self.nh, self.nkv, self.hd,
                                      self.dtype, self.q.device)

    def run(self, ops, plan=None, sink=None, out=None, fault=None):
        plan = plan or self.plan(ops)
        if out is None:
            out = torch.full((self.T + 2, self.nh * self.hd), 7.0, dtype=self.dtype, device=self.q.device)
        fault = ops.fault_word(self.q.device) if fault is None else fault
        ops.attn_shared(self.q, out, self.kc, self.vc, self.table, self.tok_pos, self.cu, self.seq_slot, plan,
                        self.scale, BLOCK, fault, sink=sink)
        return out

    def expected(self, sink=None):
        """(outputs, how far they may be off) in 64 bits, [T, nh * hd]."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        g = nh // nkv
        out = torch.zeros((self.T, nkv, g, hd), dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(out)
        half = torch.finfo(self.dtype).eps / 2            # a rounding to the element type
        u = 2.0 ** -24
        for b in range(self.B):
            for t in range(self.cu_host[b], self.cu_host[b + 1]):
                n = self.pos_host[t] + 1
                ids = self.table[self.slots[b], :-(-n // BLOCK)].long()
                K = self.kc[ids].transpose(1, 2).reshape(-1, nkv, hd)[:n].double().transpose(0, 1)
                V = self.vc[ids].transpose(1, 2).reshape(-1, nkv, hd)[:n].double().transpose(0, 1)
                q = self.q[t].double().view(nkv, g, hd)
                s = torch.einsum("kgd,knd->kgn", q, K) * self.scale
                # a score's error: hd products summed in 32 bits (truncated on the tensor cores: a
                # whole step each), the scaling and the exponential's argument and result
                size = torch.einsum("kgd,knd->kgn", q.abs(), K.abs()) * self.scale
                ds = (2 * (hd + 4) * u * size.amax(-1, keepdim=True) + 8 * u * s.abs().amax(-1, keepdim=True)
                      + 16 * u)
                if sink is not None:
                    s = torch.cat([s, sink.double().view(nkv, g, 1)], dim=-1)
                p = torch.softmax(s, dim=-1)[..., :n]
                o = torch.einsum("kgn,knd->kgd", p, V)
                a = torch.einsum("kgn,knd->kgd", p, V.abs())
                # the probabilities' rounding, numerator and denominator off by ds each, n additions,
                # the result's rounding
                out[t], tol[t] = o, a * ((half if self.dtype == torch.bfloat16 else 0.0) + 2 * ds
                                         + 2 * (n + 8) * u) + half * o.abs() + 1e-30
        return out.view(self.T, -1), tol.view(self.T, -1)

    def check(self, ops, plan=None, sink=None):
        out = self.run(ops, plan, sink)
        want, tol = self.expected(sink)
        off = (out[:self.T].double() - want).abs()
        assert torch.isfinite(out).all()
        assert (off <= tol).all(), f"off by up to {(off / tol).max().item():.3g} of what is allowed"
        assert (out[self.T:] == 7.0).all()                 # rows behind the last token stay as they were
        return out
