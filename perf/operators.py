"""The measured cases of the codebook operators: the feature lookup `embedding` with its gradient, and
`dropout` from a counter-based generator, alone and inside the lookup.

A compact scene keeps a codebook [V, C] and one codeword id per gaussian instead of an [N, C] feature
table.  A view looks its features up (scaled), a training step also sums the blend's feature gradient
by codeword.  Dropout regularises the features, or a rendered feature image, with a mask that both
directions draw anew from (seed, offset) and that is never stored.

The scene sizes are the benchmark's (4,096, 100,000 and 1,180,000 gaussians, a 979x546 view, C = 32 to
512); codebook sizes and ids are generic.

The dropout mask is defined by Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
as easy as 1, 2, 3", 2011).  Element e (row-major; the row number when whole rows are dropped) takes
half e % 8 (low half first) of the four words of counter (e // 8, offset) under key seed, and is
dropped when that 16-bit number is below T = round(65536 p); the others are scaled by
65536 / (65536 - T).
"""
import math
import os
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "high-dimensional-splatting_b200")
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
LOW32 = 0xFFFFFFFF
MOST_VALUES = 1_180_000 * 512  # the largest listed case


def _lookup(name, n, c, v, **more):
    case = {"name": name, "op": "lookup", "n": n, "c": c, "v": v, "table": "float32", "out": "float32",
            "ids": "int64", "spread": 1, "padding": False, "scale": 1.0, "p": 0.0, "train": False}
    case.update(more)
    return case


def _dropout(name, n, c, **more):
    case = {"name": name, "op": "dropout", "n": n, "c": c, "dtype": "float32", "p": 0.1, "rows": False, "train": True}
    case.update(more)
    return case


def listed():
    return [
        # The smallest scene's features for one view: latency.
        _lookup("lookup 4096x32", 4096, 32, 256),
        # Serving a view of the benchmark scene at the widest features.
        _lookup("lookup 1.18Mx512", 1_180_000, 512, 8192, ids="int32"),
        # The same scene from a codebook stored in bf16, looked up as the fp32 features the blend takes.
        _lookup("lookup bf16 1.18Mx128", 1_180_000, 128, 65536, table="bfloat16", ids="int32", scale=0.25),
        # Odd width and length, hidden gaussians without a codeword.
        _lookup("lookup fp16 99991x100", 99_991, 100, 5003, table="float16", out="float16", padding=True, scale=1.7),
        # One training step of the smallest scene: latency of both directions.
        _lookup("train 4096x32", 4096, 32, 256, train=True),
        # The 100K view with few codewords, some of them very popular.
        _lookup("train 100Kx32 skewed", 100_000, 32, 1024, spread=4, ids="int32", train=True),
        # The benchmark scene at C = 128, popular codewords.
        _lookup("train 1.18Mx128 skewed", 1_180_000, 128, 4096, spread=4, train=True),
        # The benchmark scene at C = 512 with feature dropout inside the lookup: the largest.
        _lookup("train 1.18Mx512 dropout", 1_180_000, 512, 8192, ids="int32", p=0.1, train=True),
        # Tokens of a large vocabulary, scaled by sqrt(C): most rows of the table get no gradient.
        _lookup("train bf16 tokens", 16_384, 512, 131_072, table="bfloat16", out="bfloat16", spread=2,
                scale=math.sqrt(512.0), train=True),
        # Dropout on the features of the smallest scene: latency.
        _dropout("dropout 4096x32", 4096, 32),
        # Dropout on a rendered 979x546 feature image and its gradient.
        _dropout("dropout image x128", 979 * 546, 128, p=0.25),
        # Whole gaussians dropped, half precision, odd sizes, one direction.
        _dropout("dropout rows bf16", 1_000_003, 75, dtype="bfloat16", p=0.5, rows=True, train=False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    n = _log_int(rng, 256, 1_180_000)
    c = rng.choice([_log_int(rng, 1, 512), 8 * _log_int(rng, 1, 64)])
    p = rng.choice([0.0, round(rng.uniform(0.02, 0.8), 3)])
    train = rng.random() < 0.6
    if rng.random() < 0.65:
        v = min(_log_int(rng, 2, 262_144), MOST_VALUES // (4 * c))
        table = rng.choice(["float32", "float32", "bfloat16", "float16"])
        return {"op": "lookup", "n": n, "c": c, "v": v, "table": table, "out": rng.choice([table, "float32"]),
                "ids": rng.choice(["int32", "int64"]), "spread": rng.choice([1, 1, 2, 4, 12]),
                "padding": rng.random() < 0.3, "scale": round(rng.uniform(0.1, 8.0), 3), "p": p, "train": train}
    return {"op": "dropout", "n": n, "c": c, "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]),
            "p": p or 0.1, "rows": rng.random() < 0.35, "train": train}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, c = case["n"], case["c"]

    def normal(rows, dtype):
        return torch.randn(rows, c, generator=gen, device="cuda").to(getattr(torch, dtype))

    state = {"case": case, "seed": seed * 1_000_003 + 17, "offset": 5 + seed}
    if case["op"] == "lookup":
        # spread 1: every codeword alike; larger: codeword k taken with the density of u ** spread.
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) ** case["spread"]
        ids = (u * case["v"]).long().clamp_(max=case["v"] - 1)
        if case["padding"]:
            ids[torch.rand(n, generator=gen, device="cuda") < 0.1] = -1
        state["ids"] = ids.to(getattr(torch, case["ids"]))
        state["table"] = normal(case["v"], case["table"]).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = normal(n, case["out"])
    else:
        state["x"] = normal(n, case["dtype"]).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = normal(n, case["dtype"])
    return state


def _threshold(p):
    return round(65536 * p)


def _keep_scale(p):
    t = _threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def _plain_keep(count, p, seed, offset, device):
    """[count] truth values: which elements the dropout keeps."""
    q = torch.arange((count + 7) // 8, device=device, dtype=torch.int64)
    w0, w1 = q & LOW32, q >> 32
    w2, w3 = torch.full_like(q, offset & LOW32), torch.full_like(q, offset >> 32)
    k0, k1 = seed & LOW32, seed >> 32
    for _ in range(10):
        p0, p1 = w0 * PHILOX_M[0], w2 * PHILOX_M[1]  # modulo 2^64: the low 64 bits of the 32 x 32 products
        w0, w1, w2, w3 = ((p1 >> 32) & LOW32) ^ w1 ^ k0, p1 & LOW32, ((p0 >> 32) & LOW32) ^ w3 ^ k1, p0 & LOW32
        k0, k1 = (k0 + PHILOX_W[0]) & LOW32, (k1 + PHILOX_W[1]) & LOW32
    words = torch.stack([w0, w1, w2, w3], dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)
    return halves[:count] >= _threshold(p)


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "lookup":
        return _plain_lookup(case, state)
    return _plain_dropout(case, state)


def _run_own(case, state):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import hds_b200

    if case["op"] == "lookup":
        table = state["table"]
        out = hds_b200.embedding(table, state["ids"], scale=case["scale"],
                                 padding_id=-1 if case["padding"] else None, dtype=getattr(torch, case["out"]),
                                 dropout_p=case["p"], seed=state["seed"], offset=state["offset"])
        if not case["train"]:
            return out
        return out.detach(), torch.autograd.grad(out, table, state["grad"])[0]
    x = state["x"]
    out = hds_b200.dropout(x, case["p"], seed=state["seed"], offset=state["offset"], rows=case["rows"])
    if not case["train"]:
        return out
    return out.detach(), torch.autograd.grad(out, x, state["grad"])[0]


def _plain_lookup(case, state):
    table, ids, n, c = state["table"].detach(), state["ids"].long(), case["n"], case["c"]
    factor = case["scale"] * _keep_scale(case["p"])
    kept = None
    if case["p"] > 0:
        kept = _plain_keep(n * c, case["p"], state["seed"], state["offset"], table.device).reshape(n, c)
    if case["padding"]:
        there = ids >= 0
        ids = torch.where(there, ids, 0)
        kept = there[:, None] if kept is None else kept & there[:, None]
    out = table.float()[ids] * factor
    if kept is not None:
        out = torch.where(kept, out, 0.0)
    out = out.to(getattr(torch, case["out"]))
    if not case["train"]:
        return out
    grad = state["grad"]
    if kept is not None:
        grad = torch.where(kept, grad, 0.0)
    # Popular codewords sum over 100,000 rows: in 64 bits.
    sums = torch.zeros(case["v"], c, dtype=torch.float64, device=table.device).index_add_(0, ids, grad.double())
    return out, (sums * factor).to(table.dtype)


def _plain_dropout(case, state):
    x, n, c = state["x"].detach(), case["n"], case["c"]
    count = n if case["rows"] else n * c
    kept = _plain_keep(count, case["p"], state["seed"], state["offset"], x.device).reshape(n, -1)
    factor = _keep_scale(case["p"])
    out = torch.where(kept, x.float() * factor, 0.0).to(x.dtype)
    if not case["train"]:
        return out
    return out, torch.where(kept, state["grad"].float() * factor, 0.0).to(x.dtype)


SIZES = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8}


def work(case):
    n, c = case["n"], case["c"]
    directions = 2 if case["train"] else 1
    if case["op"] == "dropout":
        read = 1.0 - case["p"] if case["rows"] else 1.0  # a dropped row need not be read
        return {"bytes": directions * n * c * SIZES[case["dtype"]] * (1.0 + read), "flops": directions * n * c}
    # The table's rows that are looked up, the ids, and the output; for a training step the output's
    # gradient and every row of the table's gradient.
    read = n * SIZES[case["ids"]] + min(n, case["v"]) * c * SIZES[case["table"]]
    total = read + n * c * SIZES[case["out"]]
    if case["train"]:
        total += n * c * SIZES[case["out"]] + case["v"] * c * SIZES[case["table"]]
    return {"bytes": total, "flops": directions * n * c}


def _exact_keep(count, p, seed, offset):
    """The mask once more, with the 32 x 32 products formed from 16-bit limbs and a group at a time laid
    out by halves."""
    groups = -(-count // 8)
    ctr = [torch.arange(groups, device="cuda") % 2**32, torch.arange(groups, device="cuda") // 2**32,
           torch.tensor(offset % 2**32, device="cuda").expand(groups),
           torch.tensor(offset // 2**32, device="cuda").expand(groups)]

    def product(a, b):
        low, high = a * (b % 65536), a * torch.div(b, 65536, rounding_mode="floor")
        high = high + low // 65536
        return high // 65536, (high % 65536) * 65536 + low % 65536

    for r in range(10):
        hi0, lo0 = product(PHILOX_M[0], ctr[0])
        hi1, lo1 = product(PHILOX_M[1], ctr[2])
        key = [(seed % 2**32 + r * PHILOX_W[0]) % 2**32, (seed // 2**32 + r * PHILOX_W[1]) % 2**32]
        ctr = [hi1 ^ ctr[1] ^ key[0], lo1, hi0 ^ ctr[3] ^ key[1], lo0]
    halves = torch.empty(groups, 8, dtype=torch.bool, device="cuda")
    for k in range(8):
        halves[:, k] = (ctr[k // 2] // 65536 if k % 2 else ctr[k // 2] % 65536) >= round(p * 2**16)
    return halves.view(-1)[:count]


def exact(case, seed):
    state = prepare(case, seed)
    n, c = case["n"], case["c"]
    keep_all = 1.0
    if case["p"] > 0:
        keep_all = 2.0**16 / (2**16 - round(case["p"] * 2**16)) if round(case["p"] * 2**16) < 2**16 else 0.0
    if case["op"] == "dropout":
        mask = _exact_keep(n if case["rows"] else n * c, case["p"], state["seed"], state["offset"]).view(n, -1).double()
        out = state["x"].detach().double() * mask * keep_all
        return (out, state["grad"].double() * mask * keep_all) if case["train"] else out
    rows = torch.cat([state["table"].detach().double(), torch.zeros(1, c, dtype=torch.float64, device="cuda")])
    ids = state["ids"].long()
    out = rows[ids] * (case["scale"] * keep_all)  # -1: the row of zeros
    mask = None
    if case["p"] > 0:
        mask = _exact_keep(n * c, case["p"], state["seed"], state["offset"]).view(n, c)
        out *= mask
    if not case["train"]:
        return out
    # Sums over the rows in codeword order, as differences of running sums, a block of columns at a time.
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids + 1, minlength=case["v"] + 1)
    ends = torch.cumsum(counts, 0)
    sums = torch.zeros(case["v"], c, dtype=torch.float64, device="cuda")
    for c0 in range(0, c, 32):
        g = state["grad"][:, c0:c0 + 32].double()
        if mask is not None:
            g = g * mask[:, c0:c0 + 32]
        running = torch.cumsum(g[order], 0)
        running = torch.cat([torch.zeros(1, running.shape[1], dtype=torch.float64, device="cuda"), running])
        sums[:, c0:c0 + 32] = running[ends[1:]] - running[ends[:-1]]
    return out, sums * (case["scale"] * keep_all)
