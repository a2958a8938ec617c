"""Plain implementations, in 64 bits and whole numbers, of the operators that decode several candidates of a chunk."""

import numpy as np
import torch


def attend_ref(q, k, v, lens, offsets, kp, vp, table, tails, scale=None):
    """(out, lse, spread, span) in float64 for the rows of the groups: out and lse as the operator's, spread [B, H, D] =
    sum_j p_j |v_j| and span [B, H] = scale * max_j sum_d |q_d k_jd|, which the bounds on rounding errors need."""
    B, H, D = q.shape
    HK = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    off, lens, tails = offsets.tolist(), lens.tolist(), tails.tolist()
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device=q.device)
    span = torch.zeros_like(lse)
    for g in range(len(lens)):
        for b in range(off[g], off[g + 1]):
            n = tails[b]
            pages = table[b, :-(-n // kp.shape[1])].long()
            kk, vv = (torch.cat([x[g, :lens[g]].double(), y[pages].flatten(0, 1)[:n].double()]) for x, y in ((k, kp), (v, vp)))
            if not len(kk):
                continue
            qq = q[b].double().view(HK, H // HK, D)
            z = torch.einsum("hrd,nhd->hrn", qq, kk) * scale
            p = torch.softmax(z, -1)
            out[b] = torch.einsum("hrn,nhd->hrd", p, vv).reshape(H, D)
            spread[b] = torch.einsum("hrn,nhd->hrd", p, vv.abs()).reshape(H, D)
            lse[b] = torch.logsumexp(z, -1).reshape(H)
            span[b] = (torch.einsum("hrd,nhd->hrn", qq.abs(), kk.abs()) * scale).amax(-1).reshape(H)
    return out, lse, spread, span


def attend_bounds(out, spread, span, n, D, dtype):
    """How far out and lse may be off.  u = eps / 2 of the type, e = 2^-24 of float32 (2^-23 where a sum may truncate).

    Scores: products of two 16-bit values are exact in float32; D of them are summed, so a score is off by at most
    (D + 2) 2^-23 span, and times log2(e), minus the maximum (|z| <= span): another 4 2^-24 span.  exp2 is off by 2^-21
    relative.  So every p is off by delta = (D + 4) 2^-23 span + 2^-21 relative, and the sum of them by no more.  Only the
    product with V takes p rounded to the type (u): 2 (delta + u) at most for p_j / sum p; the log of the sum is off by delta,
    and 2^-20 for the joins and the log.  The n products are summed in chains of at most n / 16 + 64 float32 additions (a
    matrix instruction takes 16 positions at least one at a time: n / 16 + 16 steps, then the joins), (n / 16 + 64) 2^-23 of
    spread, twice (values and sum).  The result is rounded once: u |out|."""
    u = torch.finfo(dtype).eps / 2
    delta = (D + 4) * 2.0 ** -23 * span + 2.0 ** -21
    chain = 2 * (n / 16 + 64) * 2.0 ** -23
    # a value below the type's smallest normal is off by up to half its smallest step
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (2 * (delta[..., None] + u) + chain) * spread * 1.01 + u * out.abs() + small, delta + chain + 2.0 ** -20


class PoolRef:
    """The pages' bookkeeping and contents, one step at a time, on numpy arrays."""

    def __init__(self, pages):
        self.k, self.v = pages.k.cpu().float().numpy().copy(), pages.v.cpu().float().numpy().copy()
        self.table, self.lens, self.refs = (t.cpu().numpy().copy() for t in (pages.table, pages.lens, pages.refs))
        self.page = pages.page

    def held(self, row):
        return [int(p) for p in self.table[row] if p >= 0]

    def extend(self, count, rows=None):
        rows = list(range(len(self.lens))) if rows is None else list(rows)
        free, seen = [int(p) for p in np.flatnonzero(self.refs == 0)], set()
        at, page, slot = 0, np.full((len(rows), count), -1), np.full((len(rows), count), -1)
        for i, row in enumerate(rows):
            if not 0 <= row < len(self.lens) or row in seen or self.lens[row] + count > self.table.shape[1] * self.page:
                continue
            seen.add(row)
            old = -(-int(self.lens[row]) // self.page)
            need = -(-(int(self.lens[row]) + count) // self.page) - old
            first, at = at, at + need
            if need and at > len(free):
                continue
            self.table[row, old:old + need] = free[first:at]
            self.refs[free[first:at]] = 1
            for j in range(count):
                pos = int(self.lens[row]) + j
                page[i, j], slot[i, j] = self.table[row, pos // self.page], pos % self.page
            self.lens[row] += count
        return page, slot

    def fork(self, src, dst):
        old_table, old_lens = self.table.copy(), self.lens.copy()
        old_k, old_v = self.k.copy(), self.v.copy()
        free, seen, at = [int(p) for p in np.flatnonzero(self.refs == 0)], set(), 0
        for s, d in zip(src, dst):
            if not (0 <= d < len(self.lens)) or d in seen:
                continue
            seen.add(d)
            if not 0 <= s < len(self.lens) or s == d:
                continue
            full, part = divmod(int(old_lens[s]), self.page)
            fresh = []
            if part:
                at += 1
                if at > len(free):
                    continue
                fresh = [free[at - 1]]
                last = old_table[s, full]
                self.k[:, fresh[0], :part], self.v[:, fresh[0], :part] = old_k[:, last, :part], old_v[:, last, :part]
            for p in old_table[d][old_table[d] >= 0]:
                self.refs[p] -= 1
            now = [int(p) for p in old_table[s, :full]] + fresh
            for p in now:
                self.refs[p] += 1
            self.table[d] = -1
            self.table[d, :len(now)] = now
            self.lens[d] = old_lens[s]

    def free(self, rows=None):
        for row in range(len(self.lens)) if rows is None else rows:
            for p in self.held(row):
                self.refs[p] -= 1
            self.table[row], self.lens[row] = -1, 0

    def compact(self):
        used = np.flatnonzero(self.refs > 0)
        live = len(used)
        movers, holes = used[used >= live], np.flatnonzero(self.refs[:live] == 0)
        for a, b in zip(movers, holes):
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        return live

    def check(self, pages):
        for name in ("table", "lens", "refs"):
            np.testing.assert_array_equal(getattr(pages, name).cpu().numpy(), getattr(self, name), err_msg=name)
        np.testing.assert_array_equal(pages.k.cpu().float().numpy(), self.k)
        np.testing.assert_array_equal(pages.v.cpu().float().numpy(), self.v)


def penalize_ref(logits, history=None, lens=None, repetition=None, presence=None, frequency=None, bias=None, mask=None,
                 mask_index=None):
    """float64 [B, V] of CPU tensors."""
    x = logits.double().clone()
    B, V = x.shape
    for b in range(B):
        if history is not None:
            h = history[b, :int(lens[b])]
            c = torch.bincount(h[(h >= 0) & (h < V)], minlength=V).double()
            seen = c > 0
            if repetition is not None:
                r = float(repetition[b])
                x[b] = torch.where(seen, torch.where(x[b] > 0, x[b] / r, x[b] * r), x[b])
            x[b] = torch.where(seen, x[b] - c * float(0 if frequency is None else frequency[b])
                               - float(0 if presence is None else presence[b]), x[b])
        if bias is not None:
            x[b] += (bias if bias.dim() == 1 else bias[b]).double()
        if mask is not None:
            m = int(mask_index[b]) if mask_index is not None else 0 if mask.shape[0] == 1 else b
            if m >= 0:
                words = mask[m].numpy().astype(np.uint32)
                bits = (words[:, None] >> np.arange(32, dtype=np.uint32)) & 1
                x[b, torch.from_numpy(bits.reshape(-1)[:V] == 0)] = float("-inf")
    return x
