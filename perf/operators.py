"""Workloads of the operators beside the optimizer step: the embedding lookup, its gradient and dropout.

Every case is a dict of plain values.  With ``own`` false, ``run`` computes the operator from elementary
torch operations in 32 bits (64 for f64 tensors) and rounds once; with ``own`` true it makes the calls a
training program makes of ``nabla_amd.ops``.  ``exact`` gives the same results in 64 bits, computed apart.

Definitions
  embedding       out[t] = add[t] + scale * table[ids[t]]; an id outside the table stands for a row of zeros
  embedding_grad  grad[v] (+)= scale * sum of grad_out[t] over the t with ids[t] == v, in ascending t;
                  ids outside the table contribute nothing, whatever their rows of grad_out hold
  dropout         out[e] = residual[e] + (kept(e) ? x[e] * 65536 / (65536 - thr) : 0), thr = floor(65536 p + 1/2);
                  element e = row * cols + col is dropped if 16 bits of Philox4x32-10 (key: the seed; counter:
                  e / 8, site, low and high half of the step) are below thr: half e % 2 of word e % 8 / 2
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}


def listed():
    return [
        # serving: the input row of the one token that a decoding step feeds back (8B shapes)
        {"name": "lookup_one_token", "op": "embedding", "dtype": "bf16", "rows": 128256, "cols": 4096, "ids": 1,
         "pad": 0.0, "scale": 1.0, "add": False, "wide_ids": True},
        # a GPT-2-small batch of eight sequences: token rows on top of the position rows, f32
        {"name": "lookup_on_positions", "op": "embedding", "dtype": "f32", "rows": 50257, "cols": 768, "ids": 8192,
         "pad": 0.0, "scale": 1.0, "add": True, "wide_ids": True},
        # a padded batch of the 1.1B shapes whose embeddings are scaled by the square root of their width
        {"name": "lookup_padded_scaled", "op": "embedding", "dtype": "f16", "rows": 32000, "cols": 2048, "ids": 4999,
         "pad": 0.2, "scale": 45.25, "add": False, "wide_ids": False},
        # a training batch of the 8B shapes
        {"name": "lookup_large", "op": "embedding", "dtype": "bf16", "rows": 128256, "cols": 4096, "ids": 65536,
         "pad": 0.0, "scale": 1.0, "add": False, "wide_ids": True},
        # a short sequence's gradient, added to what earlier micro-batches left
        {"name": "grad_few_tokens", "op": "embedding_grad", "dtype": "bf16", "rows": 32000, "cols": 2048, "ids": 96,
         "pad": 0.0, "scale": 1.0, "accumulate": True, "grad": "bf16", "wide_ids": True},
        # GPT-2-small, eight sequences, a fresh gradient
        {"name": "grad_gpt2_batch", "op": "embedding_grad", "dtype": "f32", "rows": 50257, "cols": 768, "ids": 8192,
         "pad": 0.0, "scale": 1.0, "accumulate": False, "grad": "f32", "wide_ids": True},
        # 1.1B shapes: bf16 activations into f32 gradients, one of several padded micro-batches
        {"name": "grad_micro_batch", "op": "embedding_grad", "dtype": "bf16", "rows": 32000, "cols": 2048, "ids": 16384,
         "pad": 0.1, "scale": 1.0, "accumulate": True, "grad": "f32", "wide_ids": False},
        # an odd width: every row starts at another alignment
        {"name": "grad_odd_width", "op": "embedding_grad", "dtype": "f16", "rows": 50257, "cols": 771, "ids": 5003,
         "pad": 0.25, "scale": 27.75, "accumulate": False, "grad": "f16", "wide_ids": True},
        # a training batch of the 8B shapes, a fresh gradient
        {"name": "grad_large", "op": "embedding_grad", "dtype": "bf16", "rows": 128256, "cols": 4096, "ids": 65536,
         "pad": 0.0, "scale": 1.0, "accumulate": False, "grad": "bf16", "wide_ids": True},
        # one short sequence of GPT-2-small's width
        {"name": "dropout_small", "op": "dropout", "dtype": "bf16", "rows": 32, "cols": 768, "p": 0.1,
         "residual": False, "backward": False},
        # a block's output dropped and added to the residual stream, GPT-2-small, eight sequences
        {"name": "dropout_residual", "op": "dropout", "dtype": "f32", "rows": 8192, "cols": 768, "p": 0.1,
         "residual": True, "backward": False},
        # the gradient of a large batch's dropout: the same mask again, from the counter
        {"name": "dropout_grad_large", "op": "dropout", "dtype": "bf16", "rows": 32768, "cols": 4096, "p": 0.05,
         "residual": False, "backward": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("embedding", "embedding_grad", "embedding_grad", "dropout"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32", "f32", "f64"))
    limit = {"f64": 1 << 26, "f32": 1 << 27}.get(dtype, 1 << 28)  # elements, so that no draw costs more than the largest
    cols = _log(rng, 48, 8192)
    if rng.random() < 0.7:
        cols = max(8, cols // 8 * 8)
    if op == "dropout":
        rows = min(_log(rng, 1, 32768), (limit >> 1) // cols)
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "p": rng.choice((0.05, 0.1, 0.1, 0.25, 0.5)),
                "residual": rng.random() < 0.4, "backward": rng.random() < 0.4}
    case = {"op": op, "dtype": dtype, "rows": min(_log(rng, 256, 131072), limit // cols), "cols": cols,
            "ids": min(_log(rng, 1, 65536), limit // cols), "pad": rng.choice((0.0, 0.0, 0.15, 0.6)),
            "scale": rng.choice((1.0, 1.0, 8.0, 0.625)), "wide_ids": rng.random() < 0.6}
    if op == "embedding":
        case["add"] = rng.random() < 0.4
    else:
        case["accumulate"] = rng.random() < 0.5
        case["grad"] = "f32" if dtype != "f64" and rng.random() < 0.4 else dtype
    return case


def _ids(case, gen):
    """Token ids as text has them: log-uniform over the ranks (a few rows hold most of the batch), the
    ranks spread over the table; a share of -1 stands for padding."""
    n, rows = case["ids"], case["rows"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)
    ids = (rank * 1000003 + 17) % rows
    padded = torch.rand(n, generator=gen, device="cuda") < case["pad"]
    return torch.where(padded, -1, ids).to(torch.int64 if case["wide_ids"] else torch.int32)


def _randn(gen, rows, cols, dtype, scale=1.0):
    x = torch.empty(rows, cols, device="cuda", dtype=torch.float32).normal_(0.0, scale, generator=gen)
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    rows, cols, dtype = case["rows"], case["cols"], case["dtype"]
    if case["op"] == "embedding":
        s["ids"] = _ids(case, gen)
        s["table"] = _randn(gen, rows, cols, dtype, 0.02)
        s["out"] = torch.empty(case["ids"], cols, device="cuda", dtype=DTYPES[dtype])
        s["add"] = _randn(gen, case["ids"], cols, dtype, 0.02) if case["add"] else None
    elif case["op"] == "embedding_grad":
        s["ids"] = _ids(case, gen)
        s["grad_out"] = _randn(gen, case["ids"], cols, dtype)
        s["grad"] = _randn(gen, rows, cols, case["grad"]) if case["accumulate"] else \
            torch.empty(rows, cols, device="cuda", dtype=DTYPES[case["grad"]])
    else:
        s["x"] = _randn(gen, rows, cols, dtype)
        s["residual"] = _randn(gen, rows, cols, dtype) if case["residual"] else None
        s["out"] = torch.empty_like(s["x"])
        s["seed"], s["step"], s["site"] = 0x9E3779B97F4A7C15 ^ seed, 5_000_000_000 + seed % 1000, 7
    if own:  # what a training program keeps for the whole run
        from nabla_amd import ops
        if case["op"] == "embedding_grad":
            s["workspace"] = ops.EmbeddingWorkspace(case["ids"], cols)
        elif case["op"] == "dropout":
            s["rng"] = ops.DropoutRng(s["seed"], s["step"])
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from nabla_amd import ops
    case = s["case"]
    if case["op"] == "embedding":
        ops.embedding(s["table"], s["ids"], s["out"], scale=case["scale"], add=s["add"])
        return s["out"]
    if case["op"] == "embedding_grad":
        ops.embedding_grad(s["grad_out"], s["ids"], s["grad"], s["workspace"], scale=case["scale"],
                           accumulate=case["accumulate"])
        return s["grad"]
    if case["backward"] and s["residual"] is None:
        ops.dropout_grad(s["x"], case["p"], s["rng"], s["site"], s["out"])
    else:  # (a gradient that is added to another branch's is the same call, with that as residual)
        ops.dropout(s["x"], case["p"], s["rng"], s["site"], s["out"], residual=s["residual"])
    return s["out"]


def _plain(s):
    case = s["case"]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32
    if case["op"] == "embedding":
        ids = s["ids"].long()
        valid = (ids >= 0) & (ids < case["rows"])
        row = s["table"][torch.where(valid, ids, 0)].to(wide) * case["scale"]
        row = torch.where(valid[:, None], row, 0.0)
        if s["add"] is not None:
            row = s["add"].to(wide) + row
        return row.to(DTYPES[case["dtype"]])
    if case["op"] == "embedding_grad":
        ids = s["ids"].long()
        valid = (ids >= 0) & (ids < case["rows"])
        total = torch.zeros(case["rows"] + 1, case["cols"], device="cuda", dtype=wide)  # the last row: padding
        total.index_add_(0, torch.where(valid, ids, case["rows"]), s["grad_out"].to(wide))
        total = total[:-1] * case["scale"]
        if case["accumulate"]:
            total = s["grad"].to(wide) + total
        s["grad"].copy_(total)
        return s["grad"]
    kept, scale = _plain_kept(s)
    y = torch.where(kept, s["x"].to(wide) * scale, 0.0)
    if s["residual"] is not None:
        y = s["residual"].to(wide) + y
    return y.to(DTYPES[case["dtype"]])


def _plain_kept(s):
    """(which elements are kept, what they are multiplied by): Philox4x32-10 in 64-bit integers."""
    case = s["case"]
    n, low = case["rows"] * case["cols"], 0xFFFFFFFF
    c0 = torch.arange((n + 7) // 8, device="cuda")
    c1, c2, c3 = s["site"], s["step"] & low, s["step"] >> 32
    k0, k1 = s["seed"] & low, s["seed"] >> 32 & low
    c1, c2, c3 = (torch.full_like(c0, c) for c in (c1, c2, c3))
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: the low and high half are what they should be
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack((c0, c1, c2, c3), 1)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    thr = int(case["p"] * 65536 + 0.5)
    return (halves >= thr).reshape(case["rows"], case["cols"]), 65536.0 / (65536 - thr)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "embedding":
        table = torch.cat((s["table"], torch.zeros_like(s["table"][:1])))  # a last row of zeros for every other id
        ids = s["ids"].long()
        row = torch.index_select(table, 0, torch.where((ids < 0) | (ids >= case["rows"]), case["rows"], ids))
        y = row.double().mul_(case["scale"])
        return y.add_(s["add"].double()) if s["add"] is not None else y
    if case["op"] == "embedding_grad":
        ids = s["ids"].long()
        at = torch.nonzero((ids >= 0) & (ids < case["rows"]))[:, 0]
        total = torch.zeros(case["rows"], case["cols"], device="cuda", dtype=torch.float64)
        total.index_put_((ids[at],), s["grad_out"][at].double() * case["scale"], accumulate=True)
        return total.add_(s["grad"].double()) if case["accumulate"] else total
    keep, thr = _exact_kept(case["rows"] * case["cols"], s["seed"], s["step"], s["site"], case["p"])
    keep = torch.from_numpy(keep).cuda().reshape(case["rows"], case["cols"])
    y = s["x"].double().mul_(65536 / (65536 - thr)).masked_fill_(~keep, 0.0)
    return y.add_(s["residual"].double()) if s["residual"] is not None else y


def _exact_kept(n, seed, step, site, p):
    """The kept elements by numpy, a million blocks at a time."""
    thr, u = math.floor(65536 * p + 0.5), np.uint64
    keep = np.empty((n + 7) // 8 * 8, dtype=bool)
    half, mask = u(32), u(0xFFFFFFFF)
    for first in range(0, len(keep) // 8, 1 << 20):
        blocks = np.arange(first, min(first + (1 << 20), len(keep) // 8), dtype=u)
        ctr = [blocks] + [np.full_like(blocks, c) for c in (site, step % 2**32, step // 2**32)]
        key = [seed % 2**32, seed // 2**32 % 2**32]
        for _ in range(10):
            even, odd = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
            ctr = [(odd >> half) ^ ctr[1] ^ u(key[0]), odd & mask, (even >> half) ^ ctr[3] ^ u(key[1]), even & mask]
            key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
        bits = np.stack(ctr, axis=1).astype("<u4").view("<u2")  # low half first
        keep[first * 8:first * 8 + bits.size] = (bits >= thr).reshape(-1)
    return keep[:n], thr


def _distinct(case):
    """How many rows of the table a batch names, on average."""
    rank = np.arange(case["rows"], dtype=np.float64)
    share = np.log1p(1.0 / (rank + 1.0)) / math.log(case["rows"] + 1)
    tokens = case["ids"] * (1.0 - case["pad"])
    return float(np.sum(-np.expm1(tokens * np.log1p(-share)))) if case["rows"] > 1 else min(1.0, tokens)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "f64": 8}
    cols, b = case["cols"], size[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * cols
        return {"bytes": n * b * (3 if case["residual"] else 2), "flops": n * (2 if case["residual"] else 1)}
    n, tokens = case["ids"], case["ids"] * (1.0 - case["pad"])
    ids = n * (8 if case["wide_ids"] else 4)
    if case["op"] == "embedding":
        return {"bytes": ids + _distinct(case) * cols * b + n * cols * b * (2 if case["add"] else 1),
                "flops": n * cols * (2 if case["add"] else 1)}
    g = size[case["grad"]]
    written = 2 * _distinct(case) * cols * g if case["accumulate"] else case["rows"] * cols * g
    return {"bytes": ids + tokens * cols * b + written, "flops": tokens * cols}
