"""Plain 64-bit forms of the paged-cache and sampling operators."""
import numpy as np
import torch

PAGE_DTYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
WORKSPACE = 8 << 20


def token_rows(pages, table_row, length, page_tokens):
    """[tokens that exist, kv_heads, head_dim] in float64: the rows of a
    sequence's first `length` tokens, those of pages outside the pool left out."""
    rows = []
    for pos in range(min(length, len(table_row) * page_tokens)):
        page = int(table_row[pos // page_tokens])
        if 0 <= page < pages.shape[0]:
            rows.append(pages[page, :, pos % page_tokens])
    if not rows:
        return pages.new_zeros((0, pages.shape[1], pages.shape[3])).double()
    return torch.stack(rows).double()


def attention(q, key_pages, value_pages, table, lengths, slots, page_tokens):
    """(out, bound): the attention of each row of q [n, q_heads, d] in float64,
    and the rounding that a kernel may add, element by element.

    A kernel may hold an operand in two parts of its page's type (or of 11
    bits), which leaves e of it out: bf16 2^-8 * 2^-8, and as much again for
    the weights; f16 2^-11 * 2^-11; f32 parts may be cut, 2^-10 * 2^-10.  A sum
    of m terms adds m * 2^-23 (sums that cut instead of rounding).  So a score
    is off by ds <= (e + d 2^-23) sum|q k| / sqrt(d), a weight by a factor
    within 1 +- 2 ds (its own score's and the maximum's), and the mean of v by
    (4 ds + e + n 2^-22) sum p|v| (numerator and denominator)."""
    e = {torch.float32: 2.0**-19, torch.float16: 2.0**-21, torch.bfloat16: 2.0**-15}[key_pages.dtype]
    n, heads, d = q.shape
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(n):
        k, v = (token_rows(p, table[slots[i]], int(lengths[i]), page_tokens) for p in (key_pages, value_pages))
        if k.shape[0] == 0:
            continue
        group = heads // k.shape[1]
        k, v = (x.repeat_interleave(group, 1) for x in (k, v))
        s = torch.einsum("hd,nhd->hn", q[i].double(), k) / d**0.5
        ds = torch.einsum("hd,nhd->hn", q[i].double().abs(), k.abs()).amax(1) / d**0.5 * (e + d * 2.0**-23)
        p = torch.softmax(s, 1)
        out[i] = torch.einsum("hn,nhd->hd", p, v)
        bound[i] = (4 * ds + e + k.shape[0] * 2.0**-22)[:, None] * torch.einsum("hn,nhd->hd", p, v.abs())
    return out, bound


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """One row's id (nan where the row is poisoned)."""
    x = np.asarray(logits, np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or not np.isfinite(x).any():
        return np.nan
    if not 0 <= temperature < np.inf or np.isnan([top_p, min_p, uniform]).any():
        return np.nan
    if temperature == 0:
        return float(np.argmax(x))
    with np.errstate(divide="ignore"):
        w = np.exp((x - x.max()) / np.float64(np.float32(temperature)))
    order = np.lexsort((np.arange(x.size), -x))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[order])))
        order = order[: max(1, int(np.searchsorted(before[:-1], np.float64(np.float32(top_p)) * before[-1], "left")))]
    order = np.sort(order[w[order] >= min(max(np.float64(np.float32(min_p)), 0.0), 1.0)])
    mass = np.cumsum(w[order])
    u = min(max(float(uniform), 0.0), 1.0 - 2.0**-24)
    return float(order[np.searchsorted(mass, u * mass[-1], "right")])
