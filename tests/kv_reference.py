"""Plain implementations, in 64 bits on the CPU, of what an attention layer runs between its products, and builders of the
batches that the tests call them with. No code of the library is used."""

from __future__ import annotations

import math

import torch

TOP = {"fp8": 448.0, "int8": 127.0}


def decode(codes: torch.Tensor, kind: str) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).double() if kind == "fp8" else codes.view(torch.int8).double()


def encode(x: torch.Tensor, kind: str) -> torch.Tensor:
    """Nearest codes, ties to even, saturating, of f64 values already divided by their scale."""
    if kind == "fp8":
        # torch rounds f32; every f64 that is not an f32 is first moved to the f32 neighbour further from the tie
        y = x.clamp(-448, 448)
        f = y.float()
        inexact = f.double() != y
        toward = torch.nextafter(f, torch.where(y > f.double(), math.inf, -math.inf).float())
        odd = (f.view(torch.int32) & 1) == 1
        f = torch.where(inexact & ~odd, toward, f)  # round to odd: a second rounding to fewer bits is then exact
        return f.to(torch.float8_e4m3fn).view(torch.uint8)
    return x.clamp(-127, 127).round().to(torch.int8).view(torch.uint8)


def power_of_two(largest: float, kind: str) -> float:
    if largest == 0:
        return 2.0**-100
    e = -100
    while largest > TOP[kind] * 2.0**e:
        e += 1
    return 2.0**e


def rotate(x, positions, frequencies, interleaved):
    """x f64 [T, heads, D]; positions int [T]; frequencies f64 [r / 2] or None."""
    if frequencies is None:
        return x
    r = 2 * frequencies.numel()
    angle = positions.double()[:, None, None] * frequencies
    c, s, y = angle.cos(), angle.sin(), x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def append(codes, scale, kind, x, starts, lengths, table, P):
    """Appends x f64 [T, heads, D], already rotated, to copies of codes [pages, heads, P, D] and scale [pages, heads]."""
    codes, scale = codes.clone(), scale.clone()
    for s, length in enumerate(lengths):
        r0, r1 = starts[s], starts[s + 1]
        first = length - (r1 - r0)
        if r0 < 0 or r1 < r0 or r1 > x.shape[0] or first < 0:
            continue
        for page in range(first // P, (length - 1) // P + 1 if r1 > r0 else first // P):
            lo, hi = max(first, page * P), min(length, page * P + P)
            p = table[s][page] if page < len(table[s]) else -1
            if not 0 <= p < codes.shape[0]:
                continue
            new = x[r0 + lo - first:r0 + hi - first]
            for h in range(codes.shape[1]):
                part, was = new[:, h], float(scale[p, h])
                want = power_of_two(float(part.abs().max()), kind) if bool(part.isfinite().all()) else math.nan
                now = want if lo == page * P or math.isnan(want) else was if math.isnan(was) else max(was, want)
                kept = lo - page * P
                if kept and now > was:
                    codes[p, h, :kept] = encode(decode(codes[p, h, :kept], kind) * (was / now), kind)
                codes[p, h, kept:hi - page * P] = 0 if math.isnan(now) else encode(part / now, kind)
                scale[p, h] = now
    return codes, scale


def attention(q, k, k_scale, v, v_scale, kind, starts, lengths, table, P, heads, scale, window):
    """q f64 [T, heads * D]. Returns the outputs [T, heads * D] and sum_j weight_j |v_j| beside them, zeros for rows of no sequence."""
    K, D = k.shape[1], k.shape[3]
    G = heads // K
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for s, length in enumerate(lengths):
        r0, r1 = starts[s], starts[s + 1]
        n = r1 - r0
        if n <= 0 or length <= 0:
            continue
        pages = table[s][:-(-length // P)]
        slot = torch.arange(length - n, length)[:, None]
        key = torch.arange(length)[None]
        seen = key <= slot
        if window:
            seen &= key > slot - window
        for h in range(K):
            kk, vv = ((decode(c[pages, h], kind) * x[pages, h].double()[:, None, None]).reshape(-1, D)[:length] for c, x in ((k, k_scale), (v, v_scale)))
            for g in range(G):
                at = slice((h * G + g) * D, (h * G + g + 1) * D)
                score = (q[r0:r1, at] @ kk.T * scale).masked_fill(~seen, -math.inf)
                score = score - score.amax(1, keepdim=True).clamp(min=-1e300)
                w = score.exp().masked_fill(~seen, 0.0)
                w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
                out[r0:r1, at], size[r0:r1, at] = w @ vv, w @ vv.abs()
    return out, size


def norm(y, h, gate, post, pre, residual_scale, block_scale, gate_sigmoid, eps):
    """f64; returns h', x and the magnitudes |residual_scale h|, |block_scale gate u| that h' is the sum of."""
    a, b = residual_scale * h, torch.zeros_like(h)
    if y is not None:
        b = y
        if post is not None:
            b = b / (b.square().mean(1, keepdim=True) + eps).sqrt() * post
        if gate is not None:
            b = b * (torch.sigmoid(gate) if gate_sigmoid else gate)
        b = block_scale * b
    x = None if pre is None else (a + b) / ((a + b).square().mean(1, keepdim=True) + eps).sqrt() * pre
    return a + b, x, a.abs(), b.abs()


class Sequences:
    """A batch: counts of new tokens and of cached ones, pages dealt in a shuffled order, spare pages and table entries besides."""

    def __init__(self, new, total, P, seed=0, spare=3, extra=2, rows_behind=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-t // P) for t in total]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n])
            at += n
        self.unused = order[at:]
        self.P, self.new, self.total = P, list(new), list(total)
        self.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        self.tokens, self.rows = self.starts[-1], self.starts[-1] + rows_behind
        width = max(need + [0]) + extra
        # what lies past a sequence's pages names no page
        self.matrix = torch.tensor([row + [-7 if i % 2 else 2**31 - 1 for i in range(width - len(row))] for row in self.table], dtype=torch.int32).reshape(len(new), width)

    def slots(self):
        return torch.tensor([t - n + i for n, t in zip(self.new, self.total) for i in range(n)] + [0] * (self.rows - self.tokens), dtype=torch.int32)


def stored(pages, heads, P, D, kind, seed):
    """Codes and scales of a cache that earlier tokens filled; what is in a slot is finite, the pages of different loudness."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((pages, heads, P, D), generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-3, 4, (pages, heads, 1, 1), generator=g).double())
    scale = torch.tensor([[power_of_two(float(x[p, h].abs().max()), kind) for h in range(heads)] for p in range(pages)], dtype=torch.float32).reshape(pages, heads)
    return encode(x / scale.double()[:, :, None, None], kind), scale
