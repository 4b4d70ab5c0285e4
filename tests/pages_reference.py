"""The cache's pages from their definition, entry by entry on the host. Test infrastructure."""
from __future__ import annotations

import torch


def fork(table, lens, refs, parents, room, page, width=0):
    """(table, lens, refs, missing, copies): copies are (from, to, tokens) of one page each."""
    pages, B = len(refs), len(table)
    W = len(table[0]) if B else width
    is_page = lambda p: 0 <= p < pages  # noqa: E731
    size = [min(max(n, 0), W * page) for n in lens]
    count = list(refs)
    for r in range(B):
        children = sum(p == r for p in parents)
        for j, p in enumerate(table[r]):
            if is_page(p):
                if children == 0:
                    count[p] -= 1
                elif j < size[r] // page:
                    count[p] += children - 1
    free = iter([p for p in range(pages) if count[p] <= 0])
    out, new_lens, copies, wanted, given, late = [], [], [], 0, [], []
    seen = set()
    for r in parents:
        if not 0 <= r < B:
            out.append([-1] * W)
            new_lens.append(0)
            continue
        full, rest = divmod(size[r], page)
        first = r not in seen
        seen.add(r)
        row = [p if first or j < full else -1 for j, p in enumerate(table[r])]
        tail = table[r][full] if rest else -1
        copied = is_page(tail) and (not first or refs[tail] > 1)
        if rest and not first and not is_page(tail):
            row[full] = tail
        have, want = full + (rest > 0), min(W, -(-(size[r] + room) // page))
        if copied and first:
            late.append(tail)
        for j in range(W):
            if (copied and j == full) or (have <= j < want and row[j] < 0):
                wanted += 1
                row[j] = next(free, -1)
                if row[j] >= 0:
                    given.append(row[j])
                    if copied and j == full:
                        copies.append((tail, row[j], -(-rest // 16) * 16))
        out.append(row)
        new_lens.append(size[r])
    for p in late:
        count[p] -= 1
    for p in given:
        count[p] = 1
    return out, new_lens, count, wanted - len(given), copies


def compact(table, refs):
    """(table, refs, moves)"""
    used = [p for p, n in enumerate(refs) if n > 0]
    holes = [p for p in range(len(used)) if refs[p] <= 0]
    moves = dict(zip([p for p in used if p >= len(used)], holes))
    new = [0] * len(refs)
    for p in used:
        new[moves.get(p, p)] = refs[p]
    return [[moves.get(p, p) for p in row] for row in table], new, list(moves.items())


def copied(cache, copies):
    """The cache after page copies (from, to, tokens)."""
    k, v, ks, vs = (x.clone() for x in cache)
    for a, b, n in copies:
        k[b, :, :n], v[b, :, :, :n], ks[b], vs[b] = cache[0][a, :, :n], cache[1][a, :, :, :n], cache[2][a], cache[3][a]
    return k, v, ks, vs


def state(rng, page, B, longest, groups, spare=4, extra=0.0):
    """(table, lens, refs, pages): rows of `groups` prompts share full pages of them; with `extra` some pages have a holder more."""
    lens = [0] * B
    order, table = list(range(100000)), [[] for _ in range(B)]
    total = 0
    take = lambda: total_iter.pop()  # noqa: E731
    plan = []
    for b in range(B):
        g = b % groups
        if b < groups:
            plan.append(rng.choice([0, 1, rng.randint(0, longest), rng.randint(0, longest // page) * page]))
        lens[b] = plan[g] if rng.random() < 0.8 else rng.randint(0, longest)
        total += -(-lens[b] // page)
    pages = total + spare
    del order
    total_iter = list(range(pages))
    rng.shuffle(total_iter)
    for b in range(B):
        n, mother = -(-lens[b] // page), table[b % groups]
        common = rng.randint(0, min(lens[b] // page, lens[b % groups] // page)) if b >= groups else 0
        table[b] = mother[:common] + [take() for _ in range(n - common)]
    width = max([len(r) for r in table] + [0]) + rng.randint(1, 3)
    table = [r + [-1] * (width - len(r)) for r in table]
    refs = [0] * pages
    for r in table:
        for p in r:
            if p >= 0:
                refs[p] += 1
    if extra:
        refs = [n + (rng.random() < extra) if n else n for n in refs]
    return table, lens, refs, pages


def cache(pages, Hkv, hd, page, g, dev):
    byte = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int32).to(torch.int8).to(dev)  # noqa: E731
    scale = lambda: torch.rand((pages, Hkv), generator=g).to(dev)  # noqa: E731
    return byte(pages, Hkv, page, hd), byte(pages, Hkv, hd, page), scale(), scale()
