"""The accuracy that paged attention claims: how much of an F32 operand its
parts leave out, and how far its sums are off.

Worst-case bounds of long sums hide a lost part, so the first test has scores
of one product each: two tokens that matter, e^(+-s) apart, and any number of
others without weight.
"""
import numpy as np
import pytest
import torch

from paged_ref import PAGE_DTYPES, WORKSPACE

U = 2.0**-24  # half a step of F32
# What the parts of an operand leave out, relative to it: three parts of BF16
# (2^-8 each), two of F16 (2^-11 each), two of TF32 (2^-11 rounded, then 2^-10
# cut), those of the page's own values too.
LEFT = {"bf16": 2.0**-24, "f16": 2.0**-22, "f32": 2.0**-21}
SHIFT = {"bf16": 0, "f16": 14, "f32": 0}  # the exponent added to weights
DIM, HEADS, KV = 64, 16, 2


def two_tokens(dtype, sequences, seed):
    """q [sequences, HEADS, DIM] with one value a row, k and v [sequences, 2, KV, DIM]."""
    g = torch.Generator().manual_seed(seed)
    t = PAGE_DTYPES[dtype][1]
    q = torch.zeros(sequences, HEADS, DIM)
    at = torch.randint(0, DIM, (sequences, KV), generator=g)  # the coordinate of each KV head
    k = torch.zeros(sequences, 2, KV, DIM)
    size = 4.0 + 5.0 * torch.rand(sequences, HEADS, generator=g)
    key = 1.0 + torch.rand(sequences, KV, generator=g) / 8
    for i in range(sequences):
        for h in range(HEADS):
            q[i, h, at[i, h * KV // HEADS]] = size[i, h]
        for h in range(KV):
            k[i, 0, h, at[i, h]], k[i, 1, h, at[i, h]] = key[i, h], -key[i, h]
    return q, k.to(t), torch.randn(sequences, 2, KV, DIM, generator=g).to(t)


def expected(dtype, q, k, v):
    """(out, bound) of the two tokens' attention, in 64 bits.

    A score carries the scale's four roundings, what the parts of q (and of an
    F32 key) leave out, and five sums in the tensor core, each cut by 2 U at
    most: its weight is off by that times |s|.  The weight itself: two
    differences in base 2, the exponential (2^-22) and two joins (an exponential
    and two roundings each), 16 U in all beside the differences.  The mean: what
    the weights' parts (and an F32 value's) leave out, five sums, the joins and
    the sum of weights, 24 U."""
    left = LEFT[dtype]
    q, k, v = (x.double() for x in (q, k, v))
    k, v = (x.repeat_interleave(HEADS // KV, 2) for x in (k, v))
    s = torch.einsum("shd,snhd->shn", q, k) / DIM**0.5
    p = torch.softmax(s, 2)
    out = torch.einsum("shn,snhd->shd", p, v)
    both = 2 if dtype == "f32" else 1
    differences = 2 * U * ((s.amax(2) - s.amin(2)) + SHIFT[dtype] * np.log(2))
    weight = s.abs().amax(2) * (both * left + 14 * U) + differences + 16 * U
    spread = torch.einsum("shn,snhd->shd", p, (v - out[:, None]).abs())
    return out, weight[:, :, None] * spread + (both * left + 24 * U) * torch.einsum("shn,snhd->shd", p, v.abs())


def parts(x, t, n):
    """What n parts of type t hold of x."""
    held = torch.zeros_like(x)
    for _ in range(n):
        held = held + (x - held).to(t).float()
    return held


@pytest.mark.parametrize("dtype,lost", [("bf16", None), ("bf16", "q"), ("bf16", "p"), ("f16", None), ("f16", "q"), ("f16", "p")])
def test_the_bound_tells_a_part_that_is_lost(dtype, lost):
    """In F32 with the kernel's parts the result is within the bound; with a
    part less, of the queries or of the weights, it is not."""
    q, k, v = two_tokens(dtype, 64, 1)
    out, bound = expected(dtype, q, k, v)
    t, n = PAGE_DTYPES[dtype][1], 3 if dtype == "bf16" else 2
    kk, vv = (x.float().repeat_interleave(HEADS // KV, 2) for x in (k, v))
    scaled = parts(q * np.float32(np.log2(np.e) / DIM**0.5), t, n - (lost == "q"))
    s = torch.einsum("shd,snhd->shn", scaled, kk)
    p = torch.exp2(s - s.amax(2, keepdim=True))
    held = parts(p * 2.0 ** SHIFT[dtype], t, n - (lost == "p")) / 2.0 ** SHIFT[dtype]
    got = torch.einsum("shn,snhd->shd", held, vv) / p.sum(2)[:, :, None]
    over = ((got.double() - out).abs() / bound).max().item()
    assert over <= 1 if lost is None else over > 1.5


def attend(dtype, q, table, lengths, keys, values, page):
    from runtime_b200 import _lib

    lib = _lib.load()
    t = lambda x: torch.as_tensor(np.asarray(x, np.int32)).cuda()  # noqa: E731
    table, lengths, q = t(table), t(lengths), q.cuda()
    keys, values = keys.cuda(), values.cuda()
    out = torch.full_like(q, 7.0)
    ws = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    st = lib.mfk_paged_gqa(out.data_ptr(), q.data_ptr(), keys.data_ptr(), values.data_ptr(), PAGE_DTYPES[dtype][0],
                           keys.shape[0], page, table.data_ptr(), table.shape[0], table.shape[1], lengths.data_ptr(), None,
                           q.shape[0], q.shape[1], keys.shape[1], q.shape[2], ws.data_ptr(), WORKSPACE,
                           torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    return out.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("length", [2, 40, 300])
def test_no_part_of_an_operand_is_lost(dtype, length):
    """Between the two tokens, those of a page that does not exist."""
    sequences, page = 64, 1
    q, k, v = two_tokens(dtype, sequences, length)
    keys, values = (x.reshape(2 * sequences, KV, 1, DIM) for x in (k, v))
    table = np.full((sequences, length), -1)
    table[:, 0], table[:, -1] = 2 * np.arange(sequences), 2 * np.arange(sequences) + 1
    out, bound = expected(dtype, q, k, v)
    got = attend(dtype, q, table, [length] * sequences, keys, values, page)
    over = ((got.double() - out).abs() / bound).max().item()
    assert over <= 1, over


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [100, 5000, 60000])
def test_error_of_the_whole_output(dtype, dim, length):
    """At most 16 U of the output's norm.  A weight's error is that of its
    score (of size 2: the roundings of scale and sums, some 3 U each way, times
    that) and of the exponential (some 2 U): about 8 U, independent from token
    to token as the values are, so the mean's is 8 U of its norm, and as much
    again is allowed.  Weights whose third BF16 part is lost are off by a
    hundred U; sums that the tensor core carries through a long sequence, by 23 U."""
    kv, heads, page = 2, 8, 16
    g = torch.Generator().manual_seed(length + dim)
    pages = -(-length // page)
    t = PAGE_DTYPES[dtype][1]
    keys, values = (torch.randn(pages, kv, page, dim, generator=g).to(t) for _ in range(2))
    q = torch.randn(1, heads, dim, generator=g) * 2
    got = attend(dtype, q, np.arange(pages)[None], [length], keys, values, page)[0].double()
    k, v = (x.double().transpose(1, 2).reshape(-1, kv, dim)[:length].repeat_interleave(heads // kv, 1) for x in (keys, values))
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), k) / dim**0.5, 1)
    want = torch.einsum("hn,nhd->hd", p, v)
    assert ((got - want).norm() / want.norm()).item() <= 16 * U
