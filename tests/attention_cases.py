"""Ragged batches for the attention tests, and their 64-bit reference.

Tolerances are derived, per output element, from the formula's own terms.
With w the softmax weights, A = sum_j w_j |v_j|, B = max_j scale * sum_e |q_e k_je|
and n the keys of the row:
 * the output's rounding to its type: u |out|, u = eps / 2 of the type;
 * the weights' rounding to the values' 16-bit type before they meet the
   values: u A (f32 outputs: f16 pairs, 2^-22 A);
 * a score's f32 dot of D products (f32 activations: f16 pairs, 2^-22 a
   product): (D + 8) 2^-23 B, twice in a normalised weight, so 2 (D + 8) 2^-23 B A;
 * exp2 and the scale's product on arguments up to B: (2^-20 + 4 B 2^-23) A;
 * sums over n keys, numerator and normaliser, in f32 in any order: 2 n 2^-24 A.
"""
import math

import numpy as np
import torch

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SENTINEL = 123.0


def cache_type(t):
    return "bf16" if t == "bf16" else "f16"


class Batch:
    """Rows, cache and metadata of one ragged batch on the GPU.

    ``new`` and ``kv``: new tokens and cached positions of each sequence.
    Unused cache slots and unused rows hold NaN."""

    def __init__(self, qmv, t, heads, kv_heads, d, new, kv=None, page=16, layout="position", pad=0, seed=0, joint=True,
                 poison=True):
        self.qmv, self.t, self.heads, self.kv_heads, self.d = qmv, t, heads, kv_heads, d
        self.new, self.kv = list(new), list(new if kv is None else kv)
        self.page, self.layout = page, layout
        self.dtype, self.id = TYPES[t]
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = len(self.new)
        self.used = sum(self.new)
        self.tokens = self.used + pad
        cols = (heads + 2 * kv_heads) * d
        extra = 0 if joint else 8
        rows = torch.randn(max(1, self.tokens), cols + extra, generator=g, device="cuda")
        rows[:, heads * d:(heads + kv_heads) * d] += torch.randn(kv_heads * d, generator=g, device="cuda")
        if poison:
            rows[self.used:] = math.nan
        self.rows = rows.to(self.dtype)
        self.ld = cols + extra
        self.q = self.rows[:, :heads * d]
        self.k = self.rows[:, heads * d:(heads + kv_heads) * d]
        self.v = self.rows[:, (heads + kv_heads) * d:cols]
        self.start = torch.tensor([0] + list(np.cumsum(self.new)), dtype=torch.int32, device="cuda")
        self.out = torch.full((max(1, self.tokens), heads * d), SENTINEL, dtype=self.dtype, device="cuda")
        ct, self.cache_id = TYPES[cache_type(t)]
        pages = [-(-x // page) for x in self.kv]
        self.width = max(pages + [1]) + 1
        self.count = sum(pages) + 2
        order = torch.randperm(self.count, generator=g, device="cuda")
        table = torch.full((n, self.width), self.count + 12345, dtype=torch.int64, device="cuda")
        at = 0
        for s, p in enumerate(pages):
            table[s, :p] = order[at:at + p]
            at += p
        self.table = table.to(torch.int32).contiguous()
        self.length = torch.tensor(self.kv, dtype=torch.int32, device="cuda")
        shape = (self.count, page, kv_heads, d) if layout == "position" else (self.count, kv_heads, page, d)
        fill = math.nan if poison else 0.0
        self.keys = torch.full(shape, fill, dtype=ct, device="cuda")
        self.values = torch.full(shape, fill, dtype=ct, device="cuda")
        kb = torch.randn(kv_heads, d, generator=g, device="cuda")
        for s in range(n):
            for x, bias in ((self.keys, kb), (self.values, 0.0)):
                c = torch.randn(self.kv[s], kv_heads, d, generator=g, device="cuda") + bias
                self.put(x, s, torch.arange(self.kv[s], device="cuda"), c.to(ct))
        if layout == "position":
            st = (page * kv_heads * d, kv_heads * d, d)
        else:
            st = (kv_heads * page * d, d, page * d)
        self.cache = qmv.PagedCache(self.keys, self.values, self.cache_id, kv_heads, d, page, self.count, st[0], st[1], st[2])

    def batch(self, max_query=None):
        return self.qmv.PagedBatch(self.start, self.length, self.table, len(self.new), self.tokens, self.width, max_query)

    def _at(self, x, s, pos):
        page = self.table[s].long()[pos // self.page]
        return (x if self.layout == "position" else x.transpose(1, 2)), page, pos % self.page

    def put(self, x, s, pos, value):
        x, page, row = self._at(x, s, pos)
        x[page, row] = value

    def get(self, x, s, n):
        x, page, row = self._at(x, s, torch.arange(n, device="cuda"))
        return x[page, row]

    def run_packed(self, stream=None, scale=0.0, out=None):
        self.qmv.packed_attention(self.id, self.heads, self.kv_heads, self.d, self.start, len(self.new), self.tokens, self.q,
                                  self.ld, self.k, self.ld, self.v, self.ld, self.out if out is None else out,
                                  self.heads * self.d, scale, stream=stream)

    def run_paged(self, stream=None, scale=0.0, max_query=None, out=None):
        self.qmv.paged_attention(self.cache, self.batch(max_query or max(self.new + [1])), self.id, self.heads, self.q, self.ld,
                                 self.out if out is None else out, self.heads * self.d, scale, stream=stream)

    def kv_of(self, s, packed):
        a, b = int(sum(self.new[:s])), int(sum(self.new[:s + 1]))
        if packed:
            return self.k[a:b].view(b - a, self.kv_heads, self.d).double(), self.v[a:b].view(b - a, self.kv_heads, self.d).double()
        return self.get(self.keys, s, self.kv[s]).double(), self.get(self.values, s, self.kv[s]).double()

    def check(self, packed, scale=0.0, skip=()):
        """Every row against the formula in 64 bits; untouched rows untouched."""
        torch.cuda.synchronize()
        worst = 0.0
        scale = scale or 1.0 / math.sqrt(self.d)
        assert torch.all(self.out[self.used:] == SENTINEL), "rows behind the last sequence were written"
        for s in range(len(self.new)):
            a, n = int(sum(self.new[:s])), self.new[s]
            if n == 0 or s in skip:
                continue
            k, v = self.kv_of(s, packed)
            got = self.out[a:a + n].double().view(n, self.heads, self.d)
            q = self.q[a:a + n].double().view(n, self.heads, self.d)
            want, tol = reference(q, k, v, scale, self.t)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (s, "NaN where the formula has none, or none where it has")
            fine = torch.isfinite(want)
            assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
            err = ((got - want).abs() / tol)[fine]
            if err.numel():
                assert float(err.max()) <= 1.0, (s, n, self.kv[s], float(err.max()))
                worst = max(worst, float(err.max()))
        return worst


def reference(q, k, v, scale, t):
    """(out, tolerance) in 64 bits: q [n, heads, d], k and v [keys, kv_heads, d];
    row i sees keys 0 .. keys - n + i.  A masked key never enters a sum."""
    n, heads, d = q.shape
    keys, kv_heads = k.shape[0], k.shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, 2.0 ** -140)
    if keys == 0:
        return out, tol
    live = torch.arange(keys, device=q.device)[None, :] <= torch.arange(n, device=q.device)[:, None] + keys - n
    u = HALF_STEP[t]
    for a in range(heads):
        h = a // (heads // kv_heads)
        s = torch.where(live, scale * (q[:, a] @ k[:, h].T), -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isinf(top) & (top < 0), 0.0, top))
        w = torch.where(live, w, 0.0)
        norm = w.sum(-1, keepdim=True)
        w = torch.where(norm > 0, w / norm, w)
        # NaN and infinities of values count only where the mask lets them
        special = ~torch.isfinite(v[:, h]).all(-1)
        o = w[:, ~special] @ v[~special, h]
        mass = w[:, ~special] @ v[~special, h].abs()
        for j in torch.nonzero(special).flatten().tolist():
            o = torch.where(live[:, j:j + 1], o + w[:, j:j + 1] * v[j, h], o)
        b = torch.where(live, scale * (q[:, a].abs() @ k[:, h].abs().T), 0.0).amax(-1, keepdim=True)
        count = live.sum(-1, keepdim=True).double()
        weight = (2.0 ** -22 if t == "f32" else u) + 2 * (d + 8) * 2.0 ** -23 * b + 2.0 ** -20 + 4 * b * 2.0 ** -23 + 2 * count * 2.0 ** -24
        out[:, a] = o
        tol[:, a] = u * o.abs() + weight * mass + 2.0 ** -140 + (2.0 ** -25 if t == "f16" else 0.0)
    return out, tol
