"""The block-scaled 8-bit operators as cases to measure: the quantiser's round trip, the
product of two sets of codes, and the product grouped by ragged lists.

A block-scaled row holds e4m3 codes and, for each block of 128 components, one scale 2**s, kept as
the byte s + 127 (E8M0). s is the smallest exponent >= -126 for which the block's largest magnitude
is at most 448 * 2**s; a block of zeros has s = 0. A component's code is value / 2**s rounded to
e4m3 (nearest, ties to even). Row pitches: the codes' the dimension rounded up to 16, the scales'
the number of blocks rounded up to 4.

``run`` computes the operators from elementary torch operations in 32 bits, or, where ``own`` is
true, by calling ``proxima_b200.blockquant``.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one query of a 768-dimensional store on its way into codes and back: latency only
        {"name": "trip one query", "op": "trip", "n": 1, "dim": 768, "type": "f32"},
        # the 1M x 128 store of the exact search, encoded once and read back
        {"name": "trip store 1M x 128", "op": "trip", "n": 1_000_000, "dim": 128, "type": "f32"},
        # an odd batch of 16-bit embeddings, the last block ragged and the rows unaligned
        {"name": "trip odd bf16", "op": "trip", "n": 100_003, "dim": 1001, "type": "bf16"},
        # one query against the 1M x 128 store
        {"name": "product one query", "op": "product", "nq": 1, "n": 1_000_000, "dim": 128, "type": "f32", "out": "f32"},
        # a small batch against a shard of 768-dimensional embeddings
        {"name": "product 16 x 500k x 768", "op": "product", "nq": 16, "n": 500_000, "dim": 768, "type": "f32", "out": "f32"},
        # odd sizes: 16-bit queries, a dimension below one block
        {"name": "product odd 37 x 100003 x 96", "op": "product", "nq": 37, "n": 100_003, "dim": 96, "type": "f16", "out": "f32"},
        # a large batch against one chunk of the 768-dimensional store, every score kept
        {"name": "product 4096 x 65536 x 768", "op": "product", "nq": 4096, "n": 65_536, "dim": 768, "type": "f32", "out": "f32"},
        # a projection of many tokens: bound by the matrix instructions
        {"name": "product 8192 x 8192 x 4096", "op": "product", "nq": 8192, "n": 8192, "dim": 4096, "type": "bf16", "out": "bf16"},
        # one token for most experts: the weights' bytes are the work
        {"name": "grouped decode 64 experts", "op": "grouped", "nq": 64, "groups": 64, "n": 2048, "dim": 1024, "even": True, "type": "bf16", "out": "bf16"},
        # many tokens over the same kind of experts
        {"name": "grouped 8192 over 32", "op": "grouped", "nq": 8192, "groups": 32, "n": 2048, "dim": 2048, "even": True, "type": "bf16", "out": "bf16"},
        # queries grouped by the inverted list they probe, lists of any length, some empty
        {"name": "grouped lists", "op": "grouped", "nq": 20_000, "groups": 500, "n": 1000, "dim": 128, "even": False, "type": "f32", "out": "f32"},
        # a few small lists: latency again
        {"name": "grouped small lists", "op": "grouped", "nq": 50, "groups": 7, "n": 100, "dim": 64, "even": False, "type": "f32", "out": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["trip", "product", "grouped"])
    kind = rng.choice(["f32", "f16", "bf16"])
    dim = _log(rng, 8, 4096)
    if op == "trip":
        return {"op": op, "n": min(_log(rng, 1, 1_000_000), 128_000_000 // dim), "dim": dim, "type": kind}
    out = rng.choice(["f32", kind])
    if op == "product":
        nq = _log(rng, 1, 8192)
        n = min(_log(rng, 1, 1_000_000), 268_000_000 // nq, 384_000_000 // dim)
        n = max(1, min(n, 270_000_000_000 // (nq * dim)))
        return {"op": op, "nq": nq, "n": n, "dim": dim, "type": kind, "out": out}
    groups = _log(rng, 1, 1000)
    nq = _log(rng, 1, 16_384)
    n = max(1, min(_log(rng, 1, 4096), 256_000_000 // (groups * dim), 30_000_000 // nq))
    return {"op": op, "nq": nq, "groups": groups, "n": n, "dim": dim, "even": rng.random() < 0.5, "type": kind, "out": out}


def _up(x, to):
    return -(-x // to) * to


def _blocks(dim):
    return -(-dim // BLOCK)


def _encode(v):
    """Elementary block encoding of rows in 32 bits: the e4m3 codes (n, blocks, 128) and the exponents (n, blocks)."""
    n, dim = v.shape
    x = torch.zeros((n, _blocks(dim) * BLOCK), dtype=torch.float32, device=v.device)
    x[:, :dim] = v
    x = x.view(n, -1, BLOCK)
    top = x.abs().amax(dim=2)
    m, e = torch.frexp(top)  # top = m * 2**e with m in [0.5, 1); 448 = 0.875 * 2**9
    s = torch.where(m <= 0.875, e - 9, e - 8)
    s = torch.where(top == 0, torch.zeros_like(s), s).clamp(min=-126)
    return torch.ldexp(x, -s[:, :, None]).to(torch.float8_e4m3fn), s


def _rows(codes, s, dim):
    return torch.ldexp(codes.to(torch.float32), s[:, :, None]).reshape(codes.shape[0], -1)[:, :dim]


def _stored(v):
    """Codes and scales of rows as the store keeps them: bytes at their pitches."""
    n, dim = v.shape
    codes, s = _encode(v)
    pitch, blocks = _up(dim, 16), _blocks(dim)
    c = torch.zeros((n, max(pitch, blocks * BLOCK)), dtype=torch.uint8, device=v.device)
    c[:, :blocks * BLOCK] = codes.view(torch.uint8).view(n, -1)
    c[:, dim:] = 0
    b = torch.zeros((n, _up(blocks, 4)), dtype=torch.uint8, device=v.device)
    b[:, :blocks] = (s + 127).to(torch.uint8)
    return c[:, :pitch].contiguous(), b


def _read(codes, scales, dim):
    """The values in 32 bits that stored rows stand for."""
    n, blocks = codes.shape[0], _blocks(dim)
    c = torch.zeros((n, blocks * BLOCK), dtype=torch.float32, device=codes.device)
    c[:, :dim] = codes[:, :dim].view(torch.float8_e4m3fn).to(torch.float32)
    s = scales[:, :blocks].to(torch.int32) - 127
    return torch.ldexp(c.view(n, blocks, BLOCK), s[:, :, None]).reshape(n, -1)[:, :dim]


def _sizes(rng, groups, total):
    """Ragged group sizes that add up to `total`, about one group in eight empty."""
    w = rng.random(groups) + 0.05
    w[rng.random(groups) < 0.125] = 0.0
    if w.sum() == 0:
        w[0] = 1.0
    edges = np.round(np.cumsum(w) / w.sum() * total).astype(np.int64)
    return np.diff(edges, prepend=0)


def _vectors(gen, n, dim, kind, device):
    """Embedding-like rows: unit length on the whole, a spread of scales along the components and a few large ones."""
    spread = torch.exp(0.7 * torch.randn(dim, generator=gen, device=device))
    v = torch.randn((n, dim), generator=gen, device=device) * spread
    return (v / math.sqrt(1.6 * dim)).to(TYPES[kind])


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dim = case["dim"]
    state = {"case": case, "q": _vectors(gen, case["n"] if case["op"] == "trip" else case["nq"], dim, case["type"], device)}
    if case["op"] == "trip":
        return state
    if case["op"] == "grouped":
        # the groups' sizes go by the case, so that the output's size does, and their order by the seed
        groups, n = case["groups"], case["n"]
        rng = np.random.default_rng(groups + case["nq"])
        nq = _sizes(rng, groups, case["nq"])
        nb = np.full(groups, n, np.int64) if case["even"] else _sizes(rng, groups, groups * n)
        order = np.random.default_rng(seed).permutation(groups)
        nq, nb = nq[order], nb[order]
        state["q_offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(nq)])).to(device)
        state["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(nb)])).to(device)
        state["most"] = int(nq.max()), int(nb.max())
        state["size"] = int((nq * nb).sum())
        rows = int(nb.sum())
    else:
        rows = case["n"]
    state["codes"], state["scales"] = _stored(_vectors(gen, rows, dim, "f32", device))
    return state


def _run_own(state):
    from proxima_b200.blockquant import BlockCodes, BlockQuantizer

    case = state["case"]
    bq = BlockQuantizer(case["dim"])
    q = bq.encode(state["q"])
    if case["op"] == "trip":
        return bq.decode(q, dtype=state["q"].dtype)
    base = BlockCodes(state["codes"], state["scales"], case["dim"])
    if case["op"] == "product":
        return bq.product(q, base, dtype=TYPES[case["out"]])
    if case["even"]:
        return bq.grouped_product(q, state["q_offsets"], base, dtype=TYPES[case["out"]])
    return bq.grouped_product(q, state["q_offsets"], base, state["offsets"], out_size=state["size"], dtype=TYPES[case["out"]])


def _run_grouped(state, q, base):
    """The ragged groups laid out as one padded batch of matrices, multiplied, and the valid entries taken out."""
    qo, bo = state["q_offsets"], state["offsets"]
    groups, dim = len(qo) - 1, q.shape[1]
    most_q, most_b = state["most"]
    row = torch.arange(len(q), device=q.device)
    g = torch.searchsorted(qo[1:].contiguous(), row, right=True)
    at = row - qo[g]
    left = torch.zeros((groups, most_q, dim), device=q.device)
    left[g, at] = q
    if state["case"]["even"]:
        right = base.view(groups, most_b, dim)
        return torch.bmm(left, right.transpose(1, 2))[g, at]
    brow = torch.arange(len(base), device=q.device)
    h = torch.searchsorted(bo[1:].contiguous(), brow, right=True)
    right = torch.zeros((groups, most_b, dim), device=q.device)
    right[h, brow - bo[h]] = base
    full = torch.bmm(left, right.transpose(1, 2))
    each = (bo[1:] - bo[:-1])[g]
    r = torch.repeat_interleave(row, each, output_size=state["size"])
    c = torch.arange(state["size"], device=q.device) - (torch.cumsum(each, 0) - each)[r]
    return full[g[r], at[r], c]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    q = _rows(*_encode(state["q"]), case["dim"])
    if case["op"] == "trip":
        return q.to(state["q"].dtype)
    base = _read(state["codes"], state["scales"], case["dim"])
    if case["op"] == "product":
        return torch.matmul(q, base.t()).to(TYPES[case["out"]])
    return _run_grouped(state, q, base).to(TYPES[case["out"]])


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    dim = case["dim"]
    row = dim + _blocks(dim)  # a stored row: codes and scales
    if case["op"] == "trip":
        n = case["n"]
        # the vectors in, the codes that the encoding leaves, the vectors out
        return {"bytes": n * (2 * dim * size[case["type"]] + row), "flops": 2 * n * dim}
    rows = case["n"] * case.get("groups", 1)
    pairs = case["nq"] * case["n"]
    return {"bytes": case["nq"] * dim * size[case["type"]] + rows * row + pairs * size[case["out"]], "flops": 2 * pairs * dim}


def _exact_rows(v):
    """The values that encoded rows stand for, from the definition in 64 bits: magnitudes on a grid of 8 steps a binade."""
    v = v.double()
    n, dim = v.shape
    pad = torch.nn.functional.pad(v, (0, _up(dim, BLOCK) - dim)).reshape(-1, BLOCK)
    top = pad.abs().max(dim=1, keepdim=True).values
    s = torch.ceil(torch.log2(top / 448.0))
    s = torch.where(top > 448.0 * torch.exp2(s), s + 1, s)  # log2 next to a whole number
    s = torch.where(top <= 448.0 * torch.exp2(s - 1), s - 1, s)
    s = torch.where(top > 0, s, torch.zeros_like(s)).clamp(min=-126)
    u = pad / torch.exp2(s)
    low = torch.frexp(u.abs())[1].double() - 1  # floor(log2 |u|) wherever u is not 0
    step = torch.exp2(low.clamp(min=-6) - 3)
    u = torch.where(u == 0, u, torch.round(u / step) * step)
    return (u * torch.exp2(s)).reshape(n, -1)[:, :dim]


def exact(case, seed):
    state = prepare(case, seed)
    q = _exact_rows(state["q"])
    if case["op"] == "trip":
        return q
    dim = case["dim"]
    b = state["codes"][:, :dim].view(torch.float8_e4m3fn).double()
    b *= torch.exp2(state["scales"].double() - 127).repeat_interleave(BLOCK, dim=1)[:, :dim]
    if case["op"] == "product":
        return q @ b.t()
    qo, bo = state["q_offsets"].tolist(), state["offsets"].tolist()
    parts = [q[qo[g]:qo[g + 1]] @ b[bo[g]:bo[g + 1]].t() for g in range(case["groups"])]
    return torch.cat(parts) if case["even"] else torch.cat([p.reshape(-1) for p in parts])
