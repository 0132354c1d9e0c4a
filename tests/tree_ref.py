"""Plain 64-bit forms of the operators over drafted trees."""
import numpy as np
import torch

from paged_ref import token_rows

U = 2.0**-24  # half a step of F32
TREE_WORKSPACE = 32 << 20
# What a kernel may leave out of a product of two operands that it holds in
# parts: three BF16 parts hold all 24 bits of an F32 value, so that BF16 pages
# leave at most 2 U out (the last part rounded), F32 pages the products of
# order 3 and more, 2 U each; two F16 parts hold 22 bits.
LEFT = {torch.float32: 2.0**-22, torch.float16: 2.0**-21, torch.bfloat16: 2.0**-22}


def ancestors(parents, first, row):
    """The places of a row's ancestors and its own, from the row up; parents None: a chain."""
    if parents is None:
        return list(range(row, -1, -1))
    path = [row]
    while 0 <= int(parents[first + path[-1]]) < path[-1]:
        path.append(int(parents[first + path[-1]]))
    return path


def random_tree(rows, rng, roots=0.1):
    """Parents of a sequence's rows: mostly near ones, some roots."""
    return [-1 if r == 0 or rng.random() < roots else int(rng.integers(max(0, r - 5), r)) for r in range(rows)]


def attention(q, key_pages, value_pages, table, lengths, offsets, parents, slots, page_tokens):
    """(out, bound) of each row of q [tokens, heads, d] in float64; rows of no
    sequence are NaN.

    With e = LEFT a score is off by ds <= (e + (d + 8) 2^-23) sum|q k| / sqrt(d) (sums
    that cut; the scale's roundings), a weight by a factor within 1 +- 2 ds (its
    own score's and the maximum's) and 2^-22 (the exponential), the mean by
    (4 ds + e + (n + 8) 2^-22) sum p|v|."""
    e = LEFT[key_pages.dtype]
    n, heads, d = q.shape
    out = torch.full((n, heads, d), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(len(offsets) - 1):
        first, rows = int(offsets[i]), int(offsets[i + 1] - offsets[i])
        start = int(lengths[i]) - rows
        slot = int(slots[i])
        reach = 0 if not 0 <= slot < len(table) else min(int(lengths[i]), table.shape[1] * page_tokens)
        there = [] if reach <= 0 else [p for p in range(reach) if 0 <= int(table[slot][p // page_tokens]) < key_pages.shape[0]]
        k, v = (token_rows(p, table[slot], reach, page_tokens) if there else None for p in (key_pages, value_pages))
        position = np.array(there)
        group = heads // key_pages.shape[1]
        for r in range(rows):
            keep = np.zeros(0, bool)
            if there:
                keep = (position < start) | np.isin(position - start, ancestors(parents, first, r))
            if not keep.any():
                out[first + r] = 0.0
                continue
            kk, vv = (x[torch.from_numpy(keep)].repeat_interleave(group, 1) for x in (k, v))
            row = q[first + r].double()
            s = torch.einsum("hd,nhd->hn", row, kk) / d**0.5
            ds = torch.einsum("hd,nhd->hn", row.abs(), kk.abs()).amax(1) / d**0.5 * (e + (d + 8) * 2.0**-23)
            p = torch.softmax(s, 1)
            out[first + r] = torch.einsum("hn,nhd->hd", p, vv)
            bound[first + r] = (4 * ds + e + (int(keep.sum()) + 8) * 2.0**-22)[:, None] * torch.einsum("hn,nhd->hd", p, vv.abs())
    return out, bound


def rotated(x, weight, epsilon, theta, positions):
    """(value, bound) of rows x [tokens, heads, d], normed (weight not None) and rotated.

    The sum of squares carries at most (d / 2 + 1) U beside the roundings of mean,
    root and quotient (its half: d / 4 + 3 U in all), the normed value two more, the
    sine and cosine one, their products and the sum two: (d / 4 + 8) U of |a| + |b|."""
    d = x.shape[2]
    half = d // 2
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(2, keepdim=True) + float(np.float32(epsilon))).sqrt() * weight.double()
    frequency = np.float32(np.power(np.float64(np.float32(theta)), -2.0 * np.arange(half) / d))
    angle = torch.from_numpy((np.asarray(positions).astype(np.float32)[:, None] * frequency).astype(np.float64))[:, None]
    a, b = x[..., :half], x[..., half:]
    value = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], 2)
    size = a.abs() + b.abs()
    return value, torch.cat([size, size], 2) * (d / 4 + 8) * U


def convolution(projection, kernel, history, offsets, parents, slots):
    """(out, bound) in float64: of width products and their gate, width + 2 roundings."""
    hidden, width = kernel.shape
    x, w = projection.double(), kernel.double()
    u = x[:, :hidden] * x[:, 2 * hidden :]
    out = torch.full((x.shape[0], hidden), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(len(offsets) - 1):
        first = int(offsets[i])
        past = history[int(slots[i])].double() if 0 <= int(slots[i]) < len(history) else torch.zeros(width - 1, hidden, dtype=torch.float64)
        for r in range(int(offsets[i + 1]) - first):
            line = [u[first + a] for a in ancestors(parents, first, r)][:width]
            line += [past[width - 2 - j] for j in range(width - len(line))]
            gate = x[first + r, hidden : 2 * hidden]
            out[first + r] = sum(line[width - 1 - j] * w[:, j] for j in range(width)) * gate
            bound[first + r] = sum((line[width - 1 - j] * w[:, j]).abs() for j in range(width)) * gate.abs() * (width + 2) * U * 1.01
    return out, bound


def accept(drafted, sampled, parents, first, rows):
    """(path, next) of a sequence."""
    path = [0]
    for r in range(1, rows):
        up = r - 1 if parents is None else int(parents[first + r])
        if up == path[-1] and drafted[first + r] == sampled[first + path[-1]]:
            path.append(r)
    return path, sampled[first + path[-1]]
