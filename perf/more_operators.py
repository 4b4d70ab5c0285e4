"""Linears with 4-bit weights and the pages of the key/value cache, as cases that can be timed and compared.

4-bit weights (the OCP microscaling format of fp4 elements): a row of K weights is K / 2 bytes of codes, weight
2 i in the low half of byte i, and K / 32 scales, one byte for each group of 32: weight = value[code] 2^(scale - 127),
value = 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the same negated. The cache of a layer is (k, v, ks, vs): int8 keys (pages,
kv heads, page, head_dim), int8 values with the tokens innermost (pages, kv heads, head_dim, page), and one fp32 scale
for each page and head of either; every layer has the same pages. refs[p] says how many places name page p (0: it is
free). A case's "kind" says which operator one pass calls:

  linear   y = x W^T (+ bias), x and y in 16 bits
  gated    silu(x G^T) * (x U^T), G the first half of the weight's rows and U the second
  fork     the rows of the page table become what "parents" says: row i continues old row parents[i], or none
           (-1). Full pages are shared. The first row of a parent keeps its last, partly filled page (unless others
           hold it too); the others get copies of it: its first slots, up to a multiple of 16, in every layer. Every row gets
           pages for `room` more tokens, the lowest free ones, row by row. Pages that nobody holds any more are free.
  compact  the pages in use move to the front: those past the number of pages in use, in their order, to the
           free ones before it
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
F64 = torch.float64
LLAMA_8B = dict(L=32, Hkv=8, hd=128)
QWEN3_1P7B = dict(L=28, Hkv=8, hd=128)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def listed():
    return [
        # one token through a small model's output projection: latency
        dict(name="linear_decode_1", kind="linear", M=1, N=2048, K=2048, bias=False, dtype="bf16"),
        # an odd decode batch through a fused qkv projection with a bias
        dict(name="linear_decode_13", kind="linear", M=13, N=6144, K=4096, bias=True, dtype="fp16"),
        # a prompt as it comes
        dict(name="linear_prompt_333", kind="linear", M=333, N=4096, K=4096, bias=False, dtype="bf16"),
        # the longest prefill's down projection
        dict(name="linear_prefill_8192", kind="linear", M=8192, N=4096, K=14336, bias=False, dtype="bf16"),
        # one token through the larger model's feed-forward block: the weights' bytes
        dict(name="gated_decode_1", kind="gated", M=1, N=14336, K=4096, dtype="bf16"),
        # a decode batch of an odd size on the smaller model
        dict(name="gated_batch_33", kind="gated", M=33, N=6144, K=2048, dtype="bf16"),
        # prefill of a whole chunk
        dict(name="gated_prefill_2048", kind="gated", M=2048, N=14336, K=4096, dtype="bf16"),
        # a step of a beam search: four prompts, four beams each
        dict(name="fork_beams_4x4", kind="fork", how="beams", groups=4, rows=4, ctx=1500, layers=32, page=64, Hkv=8, hd=128, room=1, rag=1),
        # one prompt continued 32 times
        dict(name="fork_samples_32", kind="fork", how="samples", groups=1, rows=32, ctx=2029, layers=28, page=64, Hkv=8, hd=128, room=1, rag=0),
        # between two steps of a large serving batch: some requests are done, the others get room
        dict(name="fork_serving_256", kind="fork", how="serving", groups=256, rows=1, ctx=4000, layers=4, page=16, Hkv=8, hd=128, room=1, rag=2),
        # a small pool, few layers
        dict(name="compact_150", kind="compact", pages=150, live=0.5, rows=9, layers=4, page=32, Hkv=4, hd=64, rag=3),
        # a large model's pool, half empty, before it is made smaller
        dict(name="compact_900", kind="compact", pages=900, live=0.5, rows=24, layers=32, page=64, Hkv=8, hd=128, rag=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gated", "gated", "gated", "fork", "fork", "fork", "compact", "compact"])
    if kind in ("linear", "gated"):
        M = rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 1, 8192)])
        c = dict(kind=kind, M=M, N=_log_int(rng, 33, 16384), K=32 * _log_int(rng, 2, 448), dtype=rng.choice(["bf16", "bf16", "fp16"]))
        c["M"] = min(c["M"], int(9e11 / (2 * c["N"] * c["K"] * (2 if kind == "gated" else 1))))
        if kind == "linear":
            c["bias"] = rng.random() < 0.3
        return c
    c = dict(kind=kind, layers=rng.randint(1, 36), page=rng.choice([16, 32, 64, 128]), Hkv=rng.choice([1, 2, 4, 8]),
             hd=rng.choice([32, 64, 128]), rag=rng.randint(1, 1 << 20))
    if kind == "compact":
        most = int(2e9) // (c["layers"] * 2 * c["page"] * c["Hkv"] * c["hd"])
        c.update(pages=_log_int(rng, 8, min(20000, most)), live=rng.uniform(0.05, 0.95), rows=_log_int(rng, 1, 200))
        return c
    c["how"] = rng.choice(["beams", "samples", "serving"])
    c["groups"] = 1 if c["how"] == "samples" else _log_int(rng, 1, 12) if c["how"] == "beams" else _log_int(rng, 1, 300)
    c["rows"] = 1 if c["how"] == "serving" else _log_int(rng, 1, 48 // c["groups"])
    most = int(2e9) // (c["layers"] * 2 * c["Hkv"] * c["hd"] * c["groups"])  # tokens to a group
    c["ctx"] = max(1, min(_log_int(rng, 1, 8000), most - c["rows"] * 2 * c["page"]))
    c["room"] = rng.choice([1, 1, 2, rng.randint(0, 100)])
    return c


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _weight(g, N, K):
    """Codes and scales of Gaussian weights whose rows and groups differ in size: the group's power of two brings its
    largest to [4, 8), the nearest values are taken."""
    codes, scales = [], []
    for n0 in range(0, N, 4096):
        w = _randn(g, min(4096, N - n0), K // 32, 32)
        w = w * torch.exp(0.3 * _randn(g, w.shape[0], 1, 1)) * torch.exp(0.3 * _randn(g, w.shape[0], w.shape[1], 1)) / math.sqrt(K)
        e = torch.floor(torch.log2(w.abs().amax(-1, keepdim=True).clamp(min=1e-30))) - 2
        w = w * torch.exp2(-e)
        c = torch.bucketize(w.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)) + 8 * (w < 0)
        c = c.view(w.shape[0], K // 2, 2)
        codes.append((c[..., 0] + 16 * c[..., 1]).to(torch.uint8))
        scales.append((e.squeeze(-1) + 127).to(torch.uint8))
    return torch.cat(codes), torch.cat(scales)


def _caches(g, c, pages):
    L, P, H, hd = c["layers"], c["page"], c["Hkv"], c["hd"]
    byte = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    scale = lambda: torch.exp(0.4 * _randn(g, L, pages, H)) / 30  # noqa: E731
    return byte(L, pages, H, P, hd), byte(L, pages, H, hd, P), scale(), scale()


def _held(table, pages):
    """refs of pages held by the entries of a table."""
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _fork_state(c, seed):
    """Rows of the table as forking leaves them: those of a group share the full pages of its prompt and hold the rest
    themselves."""
    rng, sizes = random.Random(seed * 1000003 + c["rag"]), random.Random(c["rag"])
    P, G, R = c["page"], c["groups"], c["rows"]
    old = 1 if c["how"] == "samples" else R
    lens, shares = [], []
    for _ in range(G):
        n = c["ctx"] if not c["rag"] else sizes.randint(max(1, c["ctx"] // 4), c["ctx"])
        lens += [n] * old
        shares.append(sizes.randint(0, n // P) if old > 1 else 0)
    need = sum(shares) + sum(-(-n // P) - shares[b // old] for b, n in enumerate(lens))
    pages = need + G * R * (2 + c["room"] // P) + 5
    order = list(range(pages))
    rng.shuffle(order)
    rows = []
    for gi in range(G):
        shared = [order.pop() for _ in range(shares[gi])]
        for b in range(gi * old, gi * old + old):
            rows.append(shared + [order.pop() for _ in range(-(-lens[b] // P) - shares[gi])])
    width = max(-(-(n + c["room"]) // P) for n in lens) + 1
    table = [r + [-1] * (width - len(r)) for r in rows]
    if c["how"] == "samples":
        parents = [0] * R
    elif c["how"] == "beams":
        parents = [gi * R + rng.randrange(R) for gi in range(G) for _ in range(R)]
    else:
        parents = [-1 if rng.random() < 0.1 else b for b in range(G)]
    return pages, table, lens, _held(table, pages), parents


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if c["kind"] in ("linear", "gated"):
        dt = TYPES[c["dtype"]]
        codes, scales = _weight(g, c["N"] * (2 if c["kind"] == "gated" else 1), c["K"])
        x = (_randn(g, c["M"], c["K"]) * torch.exp(0.5 * _randn(g, c["K"]))).to(dt)  # louder in some channels
        bias = _randn(g, c["N"]).to(dt) if c.get("bias") else None
        return dict(kind=c["kind"], x=x, codes=codes, scales=scales, bias=bias)
    if c["kind"] == "fork":
        pages, table, lens, refs, parents = _fork_state(c, seed)
        s = dict(lens=_ints(lens), parents=_ints(parents), room=c["room"])
    else:
        rng, sizes = random.Random(seed * 1000003 + c["rag"]), random.Random(c["rag"])
        pages = c["pages"]
        use = rng.sample(range(pages), max(1, int(pages * c["live"])))
        cuts = [0] + sorted(sizes.randint(0, len(use)) for _ in range(c["rows"] - 1)) + [len(use)]
        rows = [use[a:b] for a, b in zip(cuts, cuts[1:])]
        for r in rows[1:]:  # some pages of the first row belong to others too
            r[:0] = rows[0][:sizes.randint(0, min(4, len(rows[0])))]
        width = max(len(r) for r in rows) + 1
        table = [r + [-1] * (width - len(r)) for r in rows]
        refs = _held(table, pages)
        s = {}
    stack = _caches(g, c, pages)
    s.update(kind=c["kind"], stack=stack, caches=[tuple(x[i] for x in stack) for i in range(c["layers"])], table=_ints(table),
             refs=_ints(refs))
    return s


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _plain_weight(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1, 32)
    return (torch.tensor(VALUES, device=DEV)[c.long()] * torch.exp2(scales.float() - 127).unsqueeze(-1)).view(codes.shape[0], -1)


def _plain_linear(s):
    x = s["x"].float()
    y = torch.matmul(x, _plain_weight(s["codes"], s["scales"]).t())
    if s["kind"] == "gated":
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    elif s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_fork(s):
    k, v, ks, vs = s["stack"]
    table, refs, P = s["table"].long(), s["refs"].long(), s["stack"][0].shape[3]
    B, W = table.shape
    r = s["parents"].long()
    i, j = torch.arange(len(r), device=DEV), torch.arange(W, device=DEV)
    there = (r >= 0) & (r < B)
    of = r.clamp(0, B - 1)
    n = s["lens"].long()[of] * there
    full, have, want = n // P, -(-n // P), -(-(n + s["room"]) // P) * there
    first = there & ~((r[:, None] == r) & (i < i[:, None])).any(1)
    rows = table[of]
    tail = rows.gather(1, full.clamp(max=W - 1)[:, None]).squeeze(1)
    copied = there & (n % P > 0) & (tail >= 0) & (~first | (refs[tail.clamp(min=0)] > 1))
    rows = torch.where(first[:, None] | (there[:, None] & (j < full[:, None])), rows, -1)
    children = torch.zeros(B, dtype=torch.long, device=DEV).scatter_add_(0, of, there.long())[:, None]
    change = torch.where(children == 0, -1, (children - 1) * (j < (s["lens"].long() // P)[:, None])) * (table >= 0)
    refs = refs.scatter_add(0, table.clamp(min=0).flatten(), change.flatten())
    fresh = (copied[:, None] & (j == full[:, None])) | ((j >= have[:, None]) & (j < want[:, None]) & (rows < 0))
    free, order = torch.sort((refs > 0).to(torch.int32), stable=True)  # the free pages first, in their order
    rank = fresh.flatten().long().cumsum(0).view(fresh.shape) - 1
    given = torch.where(free[rank.clamp(0, len(refs) - 1)] == 0, order[rank.clamp(0, len(refs) - 1)], -1)
    rows = torch.where(fresh, given, rows)
    missing = (fresh.sum() - (free == 0).sum()).clamp(min=0)
    refs = refs.scatter_add(0, tail.clamp(min=0), -(copied & first).long())
    refs[rows[fresh & (rows >= 0)]] = 1
    row = copied.nonzero().squeeze(1)
    src, dst = tail[row], rows[row, full[row]]
    kept = (-(-(n[row] % P) // 16) * 16)[:, None] > torch.arange(P, device=DEV)
    k[:, dst] = torch.where(kept[:, None, :, None], k[:, src], k[:, dst])
    v[:, dst] = torch.where(kept[:, None, None, :], v[:, src], v[:, dst])
    ks[:, dst], vs[:, dst] = ks[:, src], vs[:, src]
    return rows.to(torch.int32), n.to(torch.int32), refs.to(torch.int32), missing.to(torch.int32).view(1), k, v, ks, vs


def _plain_compact(s):
    table, refs = s["table"].long(), s["refs"]
    at = torch.arange(len(refs), device=DEV)
    used = refs > 0
    front = at < used.sum()
    src, dst = (used & ~front).nonzero().squeeze(1), (front & ~used).nonzero().squeeze(1)
    to = at.clone()
    to[src] = dst
    moved = torch.zeros_like(refs)
    moved[to[used]] = refs[used]
    for x in s["stack"]:
        x[:, dst] = x[:, src]
    return torch.where(table >= 0, to[table.clamp(min=0)], table).to(torch.int32), moved, *s["stack"]


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    if not own:
        return {"fork": _plain_fork, "compact": _plain_compact}.get(s["kind"], _plain_linear)(s)
    w4, pages = _package()
    if s["kind"] == "linear":
        return w4.linear(s["x"], s["codes"], s["scales"], bias=s["bias"])
    if s["kind"] == "gated":
        return w4.gated(s["x"], s["codes"], s["scales"])
    if s["kind"] == "fork":
        return *pages.fork(s["caches"], s["table"], s["lens"], s["refs"], s["parents"], room=s["room"]), *s["stack"]
    return *pages.compact(s["caches"], s["table"], s["refs"]), *s["stack"]


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "useful-work-coin_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from uwc_amd import pages, w4
    return w4, pages


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] in ("linear", "gated"):
        N = c["N"] * (2 if c["kind"] == "gated" else 1)
        return dict(bytes=N * c["K"] // 2 + N * c["K"] // 32 + 2 * c["M"] * (c["K"] + c["N"]) + (2 * c["N"] if c.get("bias") else 0),
                    flops=2 * c["M"] * N * c["K"])
    token = c["layers"] * 2 * c["Hkv"] * c["hd"]
    scales = c["layers"] * 8 * c["Hkv"]
    if c["kind"] == "compact":
        rng = random.Random(c["rag"])
        use = rng.sample(range(c["pages"]), max(1, int(c["pages"] * c["live"])))
        moves = sum(p >= len(use) for p in use)
        return dict(bytes=2 * moves * (token * c["page"] + scales) + 8 * c["pages"] + 8 * len(use), flops=0)
    pages, table, lens, _, parents = _fork_state(c, 0)
    seen, moved, copies = set(), 0, 0
    for r in parents:
        if r in seen and lens[r] % c["page"]:
            moved += -(-(lens[r] % c["page"]) // 16) * 16
            copies += 1
        if r >= 0:
            seen.add(r)
    return dict(bytes=2 * (moved * token + copies * scales) + 4 * (len(table) + len(parents)) * len(table[0]) + 8 * pages, flops=0)


# ------------------------------------------------------------------ the same from the definitions, in 64 bits
def _exact_linear(c, s):
    if 2.0 * c["M"] * c["N"] * c["K"] > 4e12:
        return None
    x = s["x"].to(F64)
    value = torch.tensor([[0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0][i % 8] * (-1) ** (i // 8) for i in range(16)], dtype=F64, device=DEV)
    N, parts = s["codes"].shape[0], []
    for n0 in range(0, N, 1024):
        b = s["codes"][n0:n0 + 1024].to(torch.int32)
        w = torch.empty(b.shape[0], c["K"], dtype=F64, device=DEV)
        w[:, 0::2], w[:, 1::2] = value[b % 16], value[b // 16]
        w *= torch.pow(torch.tensor(2.0, dtype=F64, device=DEV), s["scales"][n0:n0 + 1024].to(F64) - 127).repeat_interleave(32, 1)
        parts.append(torch.matmul(x, w.t().contiguous()))
    y = torch.cat(parts, 1)
    if c["kind"] == "gated":
        return y[:, :N // 2] * torch.sigmoid(y[:, :N // 2]) * y[:, N // 2:]
    return y if s["bias"] is None else y + s["bias"].to(F64)


def _exact_fork(c, s):
    """Row by row on the host."""
    P, table, lens = c["page"], s["table"].tolist(), s["lens"].tolist()
    refs, was, parents = s["refs"].tolist(), s["refs"].tolist(), s["parents"].tolist()
    B, W = len(table), len(table[0])
    rows, n, copies, last, seen = [], [], [], [], set()
    for r in range(B):
        many = sum(p == r for p in parents)
        for j, p in enumerate(table[r]):
            if p >= 0:
                refs[p] += -1 if not many else many - 1 if j < lens[r] // P else 0
    free = [p for p in range(len(refs)) if refs[p] <= 0][::-1]
    missing = 0
    for r in parents:
        if not 0 <= r < B:
            rows.append([-1] * W)
            n.append(0)
            continue
        full, rest, begins = lens[r] // P, lens[r] % P, r not in seen
        seen.add(r)
        row = list(table[r]) if begins else table[r][:full] + [-1] * (W - full)
        old = table[r][full] if rest else -1
        if old >= 0 and (not begins or was[old] > 1):
            row[full] = -2
            if begins:
                last.append(old)
        for j in range(full, min(W, -(-(lens[r] + c["room"]) // P))):
            wanted = row[j] == -2 or (row[j] < 0 and j >= full + (rest > 0))
            if wanted:
                new = free.pop() if free else -1
                missing += new < 0
                if row[j] == -2 and new >= 0:
                    copies.append((old, new, -(-rest // 16) * 16))
                row[j] = new
        if row[full:full + 1] == [-2]:  # without room asked for, the copy is still due
            new = free.pop() if free else -1
            missing += new < 0
            if new >= 0:
                copies.append((old, new, -(-rest // 16) * 16))
            row[full] = new
        rows.append(row)
        n.append(lens[r])
    for p in last:
        refs[p] -= 1
    for r, row in zip(parents, rows):
        for j, p in enumerate(row):
            if p >= 0 and (p not in table[r]):
                refs[p] = 1
    k, v, ks, vs = (x.clone() for x in s["stack"])
    for a, b, m in copies:
        k[:, b, :, :m], v[:, b, :, :, :m], ks[:, b], vs[:, b] = k[:, a, :, :m], v[:, a, :, :, :m], ks[:, a], vs[:, a]
    return _ints(rows), _ints(n), _ints(refs), _ints([missing]), k, v, ks.to(F64), vs.to(F64)


def _exact_compact(s):
    refs = s["refs"].tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    to = {p: p for p in used if p < len(used)}
    holes = [p for p in range(len(used)) if p not in to]
    to.update(zip([p for p in used if p >= len(used)], holes))
    moved = [0] * len(refs)
    for p in used:
        moved[to[p]] = refs[p]
    table = [[to.get(p, p) for p in row] for row in s["table"].tolist()]
    out = []
    for x in s["stack"]:
        y = x.clone()
        for a, b in to.items():
            y[:, b] = x[:, a]
        out.append(y)
    return _ints(table), _ints(moved), out[0], out[1], out[2].to(F64), out[3].to(F64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("linear", "gated"):
        return _exact_linear(case, s)
    return _exact_fork(case, s) if case["kind"] == "fork" else _exact_compact(s)
