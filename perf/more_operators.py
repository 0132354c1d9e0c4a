"""The operators of drafted trees of tokens: cases, plain forms and exact values.

Four operators with which a server verifies several drafted tokens of every
sequence in one step, next to its paged caches and its models' convolutions.
``mfk_paged_append_rope`` norms and rotates the queries and keys of the drafted
rows and writes keys and values into pages, ``mfk_paged_tree_gqa`` attends with
every row to its sequence's tokens and its own ancestors, and
``mfk_tree_convolution`` (with ``mfk_tree_convolution_keep``, which moves a
history on) is the short convolution along the tree's branches.
``mfk_paged_accept`` finds the drafted rows that the model's own draws agree
with and moves their keys and values together.  ``run`` computes them in
elementary torch operations, or through the framework where ``own`` is set.

A rotation's angle is position * frequency, frequency and product rounded to 32
bits as in every rotation of this framework: caches that several of its calls
write have to agree, so the rounding belongs to the definition.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
WORKSPACE = 32 << 20
EPSILON = 1e-5
THETA = 1e6


def listed():
    return [
        # One conversation whose draft is a small tree: launch latency is all of it.
        dict(name="attention one tree", op="attention", seqs=1, past_low=249, past_high=249, rows_low=8, rows_high=8, shape="tree", q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # Conversations of every age with drafts of every size, in the framework's F32 cache type.
        dict(name="attention ragged f32", op="attention", seqs=32, past_low=0, past_high=2320, rows_low=1, rows_high=16, shape="tree", q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # A full batch with large trees.
        dict(name="attention 64 trees", op="attention", seqs=64, past_low=1000, past_high=4000, rows_low=24, rows_high=32, shape="tree", q_heads=32, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # One very long document, the small model's heads: the work is split over the length.
        dict(name="attention long f16", op="attention", seqs=1, past_low=131000, past_high=131000, rows_low=47, rows_high=47, shape="tree", q_heads=16, kv_heads=8, dim=64, page=64, dtype="f16"),
        # Prompts that go on in chunks over what the cache holds (chains), wide heads in large groups.
        dict(name="attention prompt chunks", op="attention", seqs=4, past_low=0, past_high=3000, rows_low=250, rows_high=512, shape="chain", q_heads=16, kv_heads=2, dim=128, page=24, dtype="bf16"),
        # One conversation's draft enters the cache.
        dict(name="append one tree", op="append", seqs=1, past_low=249, past_high=249, rows_low=8, rows_high=8, shape="tree", q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # The drafts of a batch.
        dict(name="append 64 trees", op="append", seqs=64, past_low=1000, past_high=4000, rows_low=24, rows_high=32, shape="tree", q_heads=32, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # Whole prompts of several lengths.
        dict(name="append prompts", op="append", seqs=7, past_low=0, past_high=100, rows_low=301, rows_high=2501, shape="chain", q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # A convolution layer of the small model over one draft.
        dict(name="convolution one tree", op="convolution", seqs=1, rows_low=8, rows_high=8, shape="tree", hidden=1024, width=3),
        # The same over a batch of large trees, the larger models' width.
        dict(name="convolution 64 trees", op="convolution", seqs=64, rows_low=24, rows_high=32, shape="tree", hidden=2048, width=3),
        # Two candidate continuations of one conversation.
        dict(name="accept one", op="accept", seqs=1, past_low=249, past_high=249, branches=2, depth=4, layers=6, kv_heads=8, dim=64, page=16, dtype="f32"),
        # Three candidates of each sequence of a large batch.
        dict(name="accept 512", op="accept", seqs=512, past_low=1, past_high=40, branches=3, depth=5, layers=6, kv_heads=8, dim=64, page=16, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "convolution", "accept"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, rng.randint(1, 80)])
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 8 * rng.randint(1, 16)])
    heads = dict(q_heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    token = kv_heads * dim * (4 if dtype == "f32" else 2)
    if op == "accept":
        seqs, branches, depth, layers = _log_int(rng, 1, 512), rng.randint(1, 6), rng.randint(1, 12), rng.randint(1, 8)
        high = rng.randint(1, 100)
        if 2 * layers * seqs * (high + branches * depth) * token > 500 << 20:
            seqs = max(1, seqs // 16)
        return dict(op=op, seqs=seqs, past_low=rng.choice([0, high]), past_high=high, branches=branches, depth=depth, layers=layers, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    shape = rng.choice(["tree", "tree", "chain"])
    if op == "convolution":
        hidden = rng.choice([1024, 2048, rng.randint(1, 2600)])
        rows = _log_int(rng, 1, 64 if shape == "tree" else 1000)
        seqs = _log_int(rng, 1, max(1, min(512, 3600000 // (hidden * rows), 4000 // rows)))
        return dict(op=op, seqs=seqs, rows_low=rng.choice([0, 1, rows]), rows_high=rows, shape=shape, hidden=hidden, width=rng.choice([3, 3, 1, 2, 4, rng.randint(5, 16)]))
    rows = _log_int(rng, 1, 64 if shape == "tree" else 512)
    seqs = _log_int(rng, 1, max(1, min(256, 2048 // rows)))
    if op == "append":
        high = _log_int(rng, 1, max(1, min(131071, (256 << 20) // (2 * token * seqs))))
        return dict(op=op, seqs=seqs, past_low=rng.choice([0, high]), past_high=high, rows_low=rng.choice([0, 1, rows]), rows_high=rows, shape=shape, **heads)
    # As many past tokens as keep the products and the bytes below the largest case's.
    most = min(131071, (256 << 20) // (2 * token * seqs), (20 << 30) // (4 * heads["q_heads"] * dim * seqs * rows))
    high = _log_int(rng, 1, max(1, most))
    return dict(op=op, seqs=seqs, past_low=rng.choice([0, high, rng.randint(0, high)]), past_high=high, rows_low=rng.choice([0, 1, rows]), rows_high=rows, shape=shape, **heads)


def _spread(low, high, n, by):
    """n numbers over [low, high], the same for every seed."""
    return [low + (((i + 1) * by % (1 << 32)) * (high - low + 1) >> 32) for i in range(n)]


def _rows(case):
    if case["op"] == "accept":
        return [1 + case["branches"] * case["depth"]] * case["seqs"]
    rows = _spread(case["rows_low"], case["rows_high"], case["seqs"], 2246822519)
    return rows if any(rows) else [1] + rows[1:]


def _past(case):
    return _spread(case["past_low"], case["past_high"], case["seqs"], 2654435761)


def _page_tables(lengths, page, generator):
    """A page table for the lengths whose pages lie in no order, and the number of pages."""
    need = np.array([-(-n // page) for n in lengths], np.int64)
    most, pages = max(1, int(need.max())), int(need.sum()) + 3
    order = torch.randperm(pages, generator=generator).numpy().astype(np.int32)
    table = np.full((len(lengths), most), -1, np.int32)
    table[np.arange(most) < need[:, None]] = order[: int(need.sum())]
    return torch.from_numpy(table).cuda(), pages


def _int(values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    numbers = np.random.RandomState(seed % (1 << 32))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gpu, device="cuda", dtype=dtype)

    s = dict(case)
    rows = _rows(case)
    total = sum(rows)
    offsets = np.concatenate([[0], np.cumsum(rows)])
    s["offsets"], s["total"], s["most_rows"] = _int(offsets), total, max(1, max(rows))
    # The trees: a row's parent is an earlier row of its sequence, mostly a near one (-1: the first row's).
    parents, depth = np.full(total, -1), np.zeros(total, np.int64)
    if case["op"] == "accept":
        at = np.arange(total) % rows[0]
        parents = np.where(at == 0, -1, np.where((at - 1) % case["depth"] == 0, 0, at - 1))
        depth = np.where(at == 0, 0, 1 + (at - 1) % case["depth"])
    else:
        chance = numbers.rand(total)
        for i, n in enumerate(rows):
            for r in range(1, n):
                back = 1 if case["shape"] == "chain" else 1 + int(chance[offsets[i] + r] ** 2 * min(r, 12))
                parents[offsets[i] + r] = r - back
                depth[offsets[i] + r] = depth[offsets[i] + r - back] + 1
    s["parents"] = _int(parents) if case.get("shape") != "chain" else None
    if case["op"] == "convolution":
        hidden, width = case["hidden"], case["width"]
        s["projection"] = normal(total, 3 * hidden)
        s["kernel"] = normal(hidden, width) * width**-0.5
        s["history"] = normal(case["seqs"], width - 1, hidden)
        s["out"], s["history_out"] = torch.empty(total, hidden, device="cuda"), torch.empty_like(s["history"])
        # The rows that were accepted: a branch from the first row to some row.
        paths, counts = np.full(total, -1), np.zeros(case["seqs"], np.int64)
        for i, n in enumerate(rows):
            branch, r = [], numbers.randint(0, n) if n else -1
            while r >= 0:
                branch.append(r)
                r = parents[offsets[i] + r]
            counts[i] = len(branch)
            paths[offsets[i] : offsets[i] + len(branch)] = branch[::-1]
        s["paths"], s["counts"] = _int(paths), _int(counts)
        return s
    past = _past(case)
    lengths = [p + n for p, n in zip(past, rows)]
    h, d, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    s["table"], pages = _page_tables(lengths, case["page"], host)
    s["starts"], s["lengths"] = _int(past), _int(lengths)
    if case["op"] == "accept":
        s["pools"] = normal(2 * case["layers"], pages, h, case["page"], d, dtype=dtype)
        # Ids of which a row's children have different ones, and draws that agree with one child as a rule.
        drafted = numbers.randint(0, 65000, total)
        sampled = numbers.randint(0, 65000, total)
        for i in range(case["seqs"]):
            branch = 1 + numbers.randint(0, case["branches"]) * case["depth"]
            length = min(case["depth"], numbers.geometric(0.25) - 1)
            for k in range(length):
                sampled[offsets[i] + (0 if k == 0 else branch + k - 1)] = drafted[offsets[i] + branch + k]
        s["drafted"], s["sampled"] = (torch.tensor(x, dtype=torch.float32, device="cuda") for x in (drafted, sampled))
        s["paths"], s["counts"] = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (total, case["seqs"]))
        s["next"] = torch.empty(case["seqs"], device="cuda")
        s["addresses"] = np.array([s["pools"][i].data_ptr() for i in range(2 * case["layers"])], np.uint64)
        return s
    s["keys"], s["values"] = (normal(pages, h, case["page"], d, dtype=dtype) for _ in range(2))
    s["q"] = normal(total, case["q_heads"] * d)
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "attention":
        # Normalised queries and keys: their scores spread as a trained model's do.
        s["q"] *= 2.0
        s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    else:
        s["k"], s["v"] = normal(total, h * d), normal(total, h * d)
        s["q_weight"], s["k_weight"] = 1.0 + normal(d) / 4, 1.0 + normal(d) / 4
        s["positions"] = _int(np.repeat(past, rows) + depth)
    return s


def _sequence_rows(s):
    """Of every row its sequence, and its place in it."""
    offsets = s["offsets"].long()
    row = torch.arange(s["total"], device="cuda")
    sequence = torch.searchsorted(offsets, row, right=True) - 1
    return sequence, row - offsets[sequence]


def _closure(s, sequence, place):
    """[sequences, rows, rows]: which rows are a row's ancestors or itself."""
    n, most = s["seqs"], s["most_rows"]
    if s["parents"] is None:
        return torch.ones(most, most, dtype=torch.bool, device="cuda").tril().expand(n, most, most)
    step = torch.zeros(n, most, most, dtype=torch.float64, device="cuda")
    has = s["parents"] >= 0
    step[sequence[has], place[has], s["parents"][has].long()] = 1.0
    step += torch.eye(most, dtype=torch.float64, device="cuda")
    return torch.linalg.matrix_power(step, most) > 0


def _attention(s):
    n, h, d, page, most = s["seqs"], s["kv_heads"], s["dim"], s["page"], s["most_rows"]
    sequence, place = _sequence_rows(s)
    table = s["table"].clamp_min(0).long()
    tokens = torch.arange(table.shape[1] * page, device="cuda")
    # A token's place among its sequence's rows: negative before the draft.
    drafted = tokens - s["starts"][:, None]
    inside = _closure(s, sequence, place).gather(2, drafted.clamp(0, most - 1)[:, None, :].expand(n, most, -1))
    seen = (inside | (drafted < 0)[:, None, :]) & (tokens < s["lengths"][:, None])[:, None, :]

    def rows(pages):  # [n, h, tokens, d]
        return pages[table].float().permute(0, 2, 1, 3, 4).reshape(n, h, -1, d)

    group = s["q_heads"] // h
    q = torch.zeros(n, most, s["q_heads"], d, device="cuda")
    q[sequence, place] = s["q"].view(-1, s["q_heads"], d)
    q = q.view(n, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(n, h, most * group, d)
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = ((q @ rows(s["keys"]).transpose(2, 3)) * d**-0.5).masked_fill_(~seen, -math.inf)
    top = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    del scores
    total = p.sum(3, keepdim=True)
    out = (p @ rows(s["values"])) / torch.where(total > 0, total, 1.0)
    out = out.view(n, h, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, -1)
    return out[sequence, place]


def _rotated(s, x, heads, weight):
    x = x.view(-1, heads, s["dim"])
    x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPSILON) * weight
    half = s["dim"] // 2
    exponent = -2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / s["dim"]
    frequency = torch.pow(torch.tensor(float(np.float32(THETA)), dtype=torch.float64, device="cuda"), exponent).float()
    angle = (s["positions"].float()[:, None] * frequency)[:, None].double()
    cosine, sine = torch.cos(angle).float(), torch.sin(angle).float()
    first, second = x[..., :half], x[..., half:]
    return torch.cat([first * cosine - second * sine, second * cosine + first * sine], 2).reshape(s["total"], -1)


def _append(s):
    sequence, place = _sequence_rows(s)
    position = s["starts"][sequence] + place
    at, off = s["table"][sequence, position // s["page"]].long(), position % s["page"]
    keys = _rotated(s, s["k"], s["kv_heads"], s["k_weight"])
    s["keys"][at, :, off] = keys.view(-1, s["kv_heads"], s["dim"]).to(s["keys"].dtype)
    s["values"][at, :, off] = s["v"].view(-1, s["kv_heads"], s["dim"]).to(s["values"].dtype)
    return _rotated(s, s["q"], s["q_heads"], s["q_weight"]), s["keys"], s["values"]


def _convolution(s):
    hidden, hist, n, most = s["hidden"], s["width"] - 1, s["seqs"], s["most_rows"]
    sequence, place = _sequence_rows(s)
    b, c, v = s["projection"].split(hidden, 1)
    # Of every sequence: its history, then its rows.
    line = torch.zeros(n, hist + most, hidden, device="cuda")
    line[:, :hist] = s["history"]
    line[sequence, hist + place] = b * v
    parents = place - 1
    if s["parents"] is not None:
        parents = torch.where(place > 0, s["parents"].long(), -1)
    # back[i]: the place in the line before place i (a history entry's is the entry before it).
    back = (torch.arange(hist + most, device="cuda") - 1).clamp_min(0).expand(n, -1).clone()
    back[sequence, hist + place] = hist + parents
    taps = [hist + place]
    for _ in range(hist):
        taps.append(back[sequence, taps[-1]])
    total = sum(line[sequence, taps[hist - j]] * s["kernel"][:, j] for j in range(hist + 1))
    # The history after the accepted rows: the last entries of the old one and theirs.
    offsets, counts = s["offsets"].long(), s["counts"].long()
    if hist == 0 or s["total"] == 0:
        return total * c, s["history"].clone()
    entry = counts[:, None] + torch.arange(hist, device="cuda")
    kept = s["paths"][(offsets[:-1, None] + entry - hist).clamp(0, s["total"] - 1)].long()
    where = torch.where(entry < hist, entry, hist + kept)
    return total * c, line[torch.arange(n, device="cuda")[:, None], where]


def _accept(s):
    n, most = s["seqs"], s["most_rows"]
    sequence, place = _sequence_rows(s)
    parents = s["parents"].view(n, most).long()
    drafted, sampled = s["drafted"].view(n, most), s["sampled"].view(n, most)
    agrees = (sampled.gather(1, parents.clamp_min(0)) == drafted) & (parents >= 0)
    # Of a row's children that agree, the first.
    twin = (parents[:, :, None] == parents[:, None, :]) & agrees[:, None, :]
    first = agrees & ~(twin & torch.ones(most, most, dtype=torch.bool, device="cuda").tril(-1)).any(2)
    first[:, 0] = True
    ancestors = _closure(s, sequence, place)
    on = (~ancestors | first[:, None, :]).all(2)
    counts = on.sum(1)
    paths = torch.where(on, torch.arange(most, device="cuda"), most).sort(1).values
    last = paths.gather(1, counts[:, None] - 1)
    position = s["starts"][:, None] + torch.stack([paths.clamp_max(most - 1), torch.arange(most, device="cuda").expand(n, -1)])
    page, off = s["table"].long()[torch.arange(n, device="cuda")[:, None], position // s["page"]], position % s["page"]
    moved = paths < most
    (from_page, to_page), (from_off, to_off) = page[:, moved], off[:, moved]
    s["pools"][:, to_page, :, to_off] = s["pools"][:, from_page, :, from_off]
    return s["pools"], torch.where(moved, paths, -1).to(torch.int32).view(-1), counts.to(torch.int32), sampled.gather(1, last)[:, 0]


def run(s):
    if not own:
        return {"attention": _attention, "append": _append, "convolution": _convolution, "accept": _accept}[s["op"]](s)
    from runtime_b200 import _lib
    from runtime_b200.backend import _check

    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream

    def at(name):
        return None if s[name] is None else s[name].data_ptr()

    if s["op"] == "convolution":
        _check(lib.mfk_tree_convolution(at("out"), at("projection"), at("kernel"), at("history"), s["seqs"], s["total"], at("offsets"), at("parents"), None, s["seqs"], s["hidden"], s["width"], stream))
        _check(lib.mfk_tree_convolution_keep(at("history_out"), at("history"), s["seqs"], at("projection"), s["total"], at("paths"), at("counts"), at("offsets"), None, s["seqs"], s["hidden"], s["width"], stream))
        return s["out"], s["history_out"]
    table = (at("table"), s["table"].shape[0], s["table"].shape[1])
    if s["op"] == "accept":
        _check(lib.mfk_paged_accept(at("paths"), at("counts"), at("next"), s["addresses"].ctypes.data, len(s["addresses"]), CODES[s["dtype"]], s["pools"].shape[1], s["page"], *table, at("drafted"), at("sampled"), s["total"], at("starts"), at("offsets"), at("parents"), None, s["seqs"], s["kv_heads"], s["dim"], stream))
        return s["pools"], s["paths"], s["counts"], s["next"]
    pages = (at("keys"), at("values"), CODES[s["dtype"]], s["keys"].shape[0], s["page"], *table)
    if s["op"] == "attention":
        _check(lib.mfk_paged_tree_gqa(at("out"), at("q"), *pages, s["total"], at("lengths"), at("offsets"), at("parents"), None, s["seqs"], s["q_heads"], s["kv_heads"], s["dim"], at("workspace"), WORKSPACE, stream))
        return s["out"]
    _check(lib.mfk_paged_append_rope(*pages, at("out"), at("q"), at("k"), at("v"), s["total"], at("q_weight"), at("k_weight"), EPSILON, THETA, at("positions"), at("starts"), at("offsets"), None, s["seqs"], s["q_heads"], s["kv_heads"], s["dim"], stream))
    return s["out"], s["keys"], s["values"]


def work(case):
    rows = _rows(case)
    total, seqs = sum(rows), case["seqs"]
    if case["op"] == "convolution":
        # Projections in, rows out, the kernel, the history in and out.
        hidden, width = case["hidden"], case["width"]
        return {"bytes": 4.0 * (4 * total * hidden + hidden * width + 2 * seqs * (width - 1) * hidden + 2 * total), "flops": 2.0 * total * hidden * (width + 1)}
    size = 4 if case["dtype"] == "f32" else 2
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "accept":
        # Some three rows of a sequence are accepted, of which two of three candidates' move.
        moved = seqs * min(3, case["depth"]) * (case["branches"] - 1) / case["branches"]
        return {"bytes": 4.0 * case["layers"] * moved * row * size + 16.0 * total + 12.0 * seqs, "flops": 0.0}
    wide = case["q_heads"] * case["dim"]
    if case["op"] == "append":
        return {"bytes": 8.0 * total * wide + 2.0 * total * row * (4 + size) + 4.0 * total + 12.0 * seqs, "flops": 8.0 * total * (wide + row)}
    past = _past(case)
    tokens = sum(past) + total
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(rows, past))
    table = sum(-(-(n + p) // case["page"]) for n, p in zip(rows, past))
    return {"bytes": 2.0 * tokens * row * size + 8.0 * total * wide + 4.0 * (table + 3 * seqs + total), "flops": 4.0 * pairs * wide}


def exact(case, seed):
    s = prepare(case, seed)
    rows = _rows(case)
    offsets = [0]
    for n in rows:
        offsets.append(offsets[-1] + n)
    parents = None if s["parents"] is None else s["parents"].tolist()

    def up(i, r):
        return r - 1 if parents is None else parents[offsets[i] + r]

    if case["op"] == "convolution":
        hidden, width = case["hidden"], case["width"]
        x, kernel = s["projection"].double(), s["kernel"].double()
        u = x[:, :hidden] * x[:, 2 * hidden :]
        out, history = torch.zeros(offsets[-1], hidden, dtype=torch.float64, device="cuda"), s["history"].double()
        after = history.clone()
        paths, counts = s["paths"].tolist(), s["counts"].tolist()
        for i, n in enumerate(rows):
            for r in range(n):
                window, at = [], r
                while len(window) < width:
                    window.append(u[offsets[i] + at] if at >= 0 else history[i, width - 1 + at])
                    at = at - 1 if at < 0 else up(i, at)
                out[offsets[i] + r] = sum(w * kernel[:, width - 1 - j] for j, w in enumerate(window)) * x[offsets[i] + r, hidden : 2 * hidden]
            kept = [history[i, j] for j in range(width - 1)] + [u[offsets[i] + paths[offsets[i] + j]] for j in range(counts[i])]
            for j in range(width - 1):
                after[i, j] = kept[len(kept) - (width - 1) + j]
        return out, after
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    past = _past(case)

    def where(i, first, count):
        position = torch.arange(first, first + count, device="cuda")
        return s["table"][i, torch.div(position, page, rounding_mode="floor")].long(), position % page

    if case["op"] == "accept":
        pools = s["pools"].clone() if case["dtype"] == "f32" else s["pools"].float()
        drafted, sampled = s["drafted"].tolist(), s["sampled"].tolist()
        last = []
        for i, n in enumerate(rows):
            path = [0]
            for r in range(1, n):
                if up(i, r) == path[-1] and drafted[offsets[i] + r] == sampled[offsets[i] + path[-1]]:
                    path.append(r)
            last.append(sampled[offsets[i] + path[-1]])
            table, off = where(i, past[i], n)
            pools[:, table[: len(path)], :, off[: len(path)]] = s["pools"][:, table[path], :, off[path]].to(pools.dtype)
        return pools, None, None, np.array(last)
    if case["op"] == "append":
        half = d // 2
        frequency = np.float32(np.power(np.float64(np.float32(THETA)), -2.0 * np.arange(half) / d))
        angle = s["positions"].cpu().numpy().astype(np.float32)[:, None] * frequency
        turn = torch.from_numpy(np.exp(1j * angle.astype(np.float64))).cuda()[:, None]
        result = []
        for x, weight, heads in ((s["q"], s["q_weight"], case["q_heads"]), (s["k"], s["k_weight"], h)):
            x = x.double().view(-1, heads, d)
            x = x / (x.pow(2).sum(2, keepdim=True) / d + EPSILON).sqrt() * weight.double()
            z = torch.complex(x[..., :half], x[..., half:]) * turn
            result.append(torch.cat([z.real, z.imag], 2).reshape(-1, heads * d))
        pages = [s["keys"].double(), s["values"].double()]
        for i, n in enumerate(rows):
            table, off = where(i, past[i], n)
            for to, x in zip(pages, (result[1], s["v"].double())):
                to[table, :, off] = x[offsets[i] : offsets[i + 1]].view(n, h, d)
        return result[0], pages[0], pages[1]
    out = torch.zeros(offsets[-1], case["q_heads"], d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(rows):
        if n == 0:
            continue
        table, off = where(i, 0, past[i] + n)
        k, v = (x[table, :, off].double().permute(1, 0, 2) for x in (s["keys"], s["values"]))
        seen = torch.zeros(n, past[i] + n, dtype=torch.bool)
        seen[:, : past[i]] = True
        for r in range(n):
            if up(i, r) >= 0:
                seen[r, past[i] :] = seen[up(i, r), past[i] :]
            seen[r, past[i] + r] = True
        seen = seen.cuda()
        group = case["q_heads"] // h
        q = s["q"][offsets[i] : offsets[i + 1]].double().view(n, h, group, d)
        for j in range(h):
            score = torch.einsum("ngd,td->gnt", q[:, j], k[j]) / math.sqrt(d)
            p = torch.softmax(score.masked_fill(~seen, -math.inf), 2)
            out[offsets[i] : offsets[i + 1], j * group : (j + 1) * group] = torch.einsum("gnt,td->ngd", p, v[j])
    return out.view(offsets[-1], -1)
