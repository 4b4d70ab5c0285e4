"""The pages of the 8-bit cache (uwc_amd.pages) on the GPU against their definition on the host: everything bit for bit."""
import random

import pytest
import torch

import pages_reference as R

pytestmark = pytest.mark.gpu


def ints(x, dev, width=None):
    t = torch.tensor(x, dtype=torch.int32, device=dev)
    return t.view(0, width) if width is not None and not len(x) else t


def caches(layers, pages, Hkv, hd, page, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return [R.cache(pages, Hkv, hd, page, g, dev) for _ in range(layers)]


def check_fork(dev, cs, page, table, lens, refs, parents, room, stride=0):
    from uwc_amd import pages as P
    before = [tuple(x.clone() for x in c) for c in cs]
    t = ints(table, dev, len(table[0]) if table else 3)
    if stride:
        wide = torch.full((t.shape[0], t.shape[1] + stride), 7, dtype=torch.int32, device=dev)
        wide[:, :t.shape[1]] = t
        t = wide[:, :t.shape[1]]
    inputs = t, ints(lens, dev), ints(refs, dev), ints(parents, dev)
    kept = [x.clone() for x in inputs]
    got = P.fork(cs, *inputs, room=room)
    want = R.fork(table, lens, refs, parents, room, page, t.shape[1])
    for name, x, y in zip(("table", "lens", "refs", "missing"), got, want):
        assert x.flatten().tolist() == [e for r in y for e in r] if name == "table" else x.tolist() == (y if name != "missing" else [y]), name
    for c, b in zip(cs, before):
        for x, y in zip(c, R.copied(b, want[4])):
            assert torch.equal(x, y)
    assert all(torch.equal(x, y) for x, y in zip(inputs, kept))
    return got


def check_compact(dev, cs, table, refs):
    from uwc_amd import pages as P
    before = [tuple(x.clone() for x in c) for c in cs]
    t, n = P.compact(cs, ints(table, dev, 3), ints(refs, dev))
    wt, wn, moves = R.compact(table, refs)
    assert t.tolist() == wt and n.tolist() == wn
    page = cs[0][0].shape[2]
    for c, b in zip(cs, before):
        for x, y in zip(c, R.copied(b, [(p, q, page) for p, q in moves])):
            assert torch.equal(x, y)
    return t, n


@pytest.mark.parametrize("page,Hkv,hd,layers", [(16, 1, 32, 1), (16, 3, 64, 2), (32, 2, 128, 3), (64, 8, 64, 1), (64, 5, 128, 2), (128, 2, 32, 2), (128, 8, 128, 1)])
@pytest.mark.parametrize("seed", range(3))
def test_fork(dev, page, Hkv, hd, layers, seed):
    rng = random.Random(seed * 100 + page + hd)
    for _ in range(4):
        B = rng.choice([1, 2, 5, 17])
        table, lens, refs, pages = R.state(rng, page, B, 5 * page, rng.randint(1, B), spare=rng.choice([0, 3, 40]), extra=rng.choice([0, 0.3]))
        cs = caches(layers, pages, Hkv, hd, page, seed, dev) if pages else None
        if not pages:
            continue
        parents = [rng.choice([rng.randrange(B), rng.randrange(B), -1]) for _ in range(rng.choice([1, B, 2 * B, 9]))]
        check_fork(dev, cs, page, table, lens, refs, parents, rng.choice([0, 1, page, 3 * page + 1]), stride=rng.choice([0, 5]))


def test_fork_of_one_prompt_many_times(dev):
    page, n = 64, 300
    table, lens, refs = [[4, 2, 9] + [-1] * 3], [150], [0] * 400
    for p in (4, 2, 9):
        refs[p] = 1
    cs = caches(2, 400, 2, 64, page, 1, dev)
    t, _, r, missing = check_fork(dev, cs, page, table, lens, refs, [0] * n, 1)
    assert r[4] == r[2] == n and r[9] == 1 and missing == 0 and len(set(t[:, 2].tolist())) == n
    check_fork(dev, cs, page, table, lens, refs, [0] * 500, 0)  # more than there are pages


def test_fork_grows_and_runs_out(dev):
    page = 16
    cs = caches(1, 6, 1, 32, page, 2, dev)
    table, lens, refs = [[0, -1, -1, -1], [5, 3, -1, -1], [-1] * 4], [16, 20, 0], [1, 0, 0, 1, 0, 1]
    check_fork(dev, cs, page, table, lens, refs, [0, 1, 2], 1)
    t, _, r, missing = check_fork(dev, cs, page, table, lens, refs, [0, 1, 2, 1], 30)
    assert missing == 2 + 2 + 2 + 3 - 3 and r.min() == 1
    check_fork(dev, cs, page, table, lens, refs, [0, 1, 2], 2 ** 31 - 1)  # as far as the table is wide
    check_fork(dev, cs, page, table, lens, refs, [-1, -1, -1], 5)  # everything ends
    check_fork(dev, cs, page, table, lens, refs, [1], 0)


def test_fork_keeps_pages_reserved_ahead(dev):
    page = 16
    cs = caches(1, 8, 1, 32, page, 3, dev)
    table, lens, refs = [[6, 1, 4, -1]], [17], [0, 1, 0, 0, 1, 0, 1, 0]  # page 4 is room that was taken before
    t, _, r, _ = check_fork(dev, cs, page, table, lens, refs, [0, 0], 20)
    assert t.tolist() == [[6, 1, 4, -1], [6, 0, 2, -1]] and r[6] == 2
    check_fork(dev, cs, page, table, lens, refs, [-1, 0], 0)


def test_fork_of_pages_that_others_hold(dev):
    """Copy on write: a prompt kept aside (its pages counted once more) is not written by the row that goes on from it."""
    page = 16
    cs = caches(2, 8, 2, 32, page, 4, dev)
    table, lens, refs = [[3, 5, -1], [3, 5, -1]], [20, 20], [0, 0, 0, 3, 0, 3, 0, 0]
    t, _, r, _ = check_fork(dev, cs, page, table, lens, refs, [0, 1, 1], 1)
    assert t.tolist() == [[3, 0, -1], [3, 1, -1], [3, 2, -1]] and r[3] == 4 and r[5] == 1


@pytest.mark.parametrize("bad", ["table", "parents", "lens"])
def test_numbers_out_of_range_touch_nothing_else(dev, bad):
    page = 16
    cs = caches(2, 9, 2, 32, page, 5, dev)
    table, lens, refs = [[0, 1, 2, -1], [3, 4, -1, -1], [5, 6, 7, -1]], [40, 17, 33], [1] * 8 + [0]
    parents = [0, 0, 1, 2]
    if bad == "table":
        table[0][2], table[1][0], table[2][1] = 9, -7, 2 ** 31 - 1
        refs[2] = refs[3] = refs[6] = 0
        lens[2] = 20
    elif bad == "parents":
        parents = [3, -2 ** 31, 2 ** 31 - 1, 1]
    else:
        lens = [-5, 10 ** 9, 2 ** 31 - 1]
    check_fork(dev, cs, page, table, lens, refs, parents, 3)


def test_fork_without_rows(dev):
    cs = caches(1, 5, 1, 32, 16, 6, dev)
    refs = [1, 0, 2, 0, 0]
    check_fork(dev, cs, 16, [], [], refs, [], 1)
    check_fork(dev, cs, 16, [], [], refs, [0, -1], 1)
    check_fork(dev, cs, 16, [[0, -1]], [3], refs, [], 1)


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 1023, 1025, 5000])
@pytest.mark.parametrize("live", [0.0, 0.1, 0.5, 0.97, 1.0])
def test_compact(dev, pages, live):
    rng = random.Random(pages + int(100 * live))
    layers, Hkv, hd, page = rng.choice([(1, 2, 32, 16), (3, 1, 64, 32), (2, 2, 32, 64)])
    cs = caches(layers, pages, Hkv, hd, page, pages, dev)
    use = rng.sample(range(pages), int(round(live * pages)))
    refs = [0] * pages
    rows = [[], use[: len(use) // 3], use[len(use) // 3:]]
    rows[0] = use[:2]
    for r in rows:
        for p in r:
            refs[p] += 1
    if pages > 4:
        free = [p for p in range(pages) if not refs[p]]
        if free:
            refs[free[0]] = -3  # as free as none
    width = max(map(len, rows)) + 2
    table = [r + [-1] * (width - len(r)) for r in rows]
    table[0][-1], table[1][-1] = pages + 3, -9
    t, n = check_compact(dev, cs, table, refs)
    check_compact(dev, cs, t.tolist(), n.tolist())  # nothing left to move


def test_many_pages_and_rows(dev):
    """Several ranges of pages, rows past 256, more layers than a launch takes."""
    rng = random.Random(9)
    table, lens, refs, pages = R.state(rng, 16, 700, 100, 90, spare=3000)
    cs = caches(1, pages, 1, 32, 16, 7, dev)
    parents = [rng.randrange(-20, 700) for _ in range(900)]
    t, l, r, _ = check_fork(dev, cs, 16, table, lens, refs, parents, 17)
    check_compact(dev, cs, t.tolist(), r.tolist())
    table, lens, refs, pages = R.state(rng, 16, 6, 100, 2)
    cs = caches(131, pages, 1, 32, 16, 8, dev)
    t, l, r, _ = check_fork(dev, cs, 16, table, lens, refs, [0, 0, 1, 3, 3, 5], 1)
    check_compact(dev, cs, t.tolist(), r.tolist())


def test_a_pool_past_two_gigabytes(dev):
    """Offsets of pages past 2^31 bytes."""
    from uwc_amd import kv, pages as P
    n, page, Hkv, hd = 17000, 128, 8, 128
    c = kv.new_cache(n, Hkv, hd, page, dev)
    c[0][n - 1], c[1][n - 1], c[2][n - 1], c[3][n - 1] = 5, 6, 7.0, 8.0
    refs = torch.zeros(n, dtype=torch.int32, device=dev)
    refs[:n - 9] = 1
    refs[n - 1] = 1
    table = torch.tensor([[n - 1, -1]], dtype=torch.int32, device=dev)
    t, _, r, _ = P.fork([c], table, ints([30], dev), refs, ints([0, 0], dev))
    assert t.tolist() == [[n - 1, -1], [n - 9, -1]]
    assert (c[0][n - 9, :, :32] == 5).all() and not c[0][n - 9, :, 32:].any() and (c[1][n - 9, :, :, :32] == 6).all()
    t, r = P.compact([c], t, r)
    assert t.tolist() == [[n - 8, -1], [n - 9, -1]] and (c[0][n - 8] == 5).all() and (c[1][n - 8] == 6).all() and (c[3][n - 8] == 8).all()


def test_streams_and_graphs(dev):
    """Captured once and replayed on other parents and counts, eager work between; two graphs do not share a workspace's contents."""
    from uwc_amd import pages as P
    page = 32
    rng = random.Random(12)
    table, lens, refs, pages = R.state(rng, page, 8, 200, 3, spare=40)
    cs = caches(3, pages, 2, 64, page, 9, dev)
    t, n, c = ints(table, dev), ints(lens, dev), ints(refs, dev)
    parents = ints([0, 0, 1, 2, 3, 3, 6, -1], dev)
    P.fork(cs, t, n, c, parents, room=1), P.compact(cs, t, c)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = P.fork(cs, t, n, c, parents, room=1)
            moved = P.compact(cs, out[0], out[2])
        graphs.append((g, out, moved))
    for i in range(4):
        new = [rng.randrange(-1, 8) for _ in range(8)]
        parents.copy_(ints(new, dev))
        before = [tuple(x.clone() for x in c_) for c_ in cs]
        g, out, moved = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        wt, wl, wr, wm, copies = R.fork(table, lens, refs, new, 1, page)
        assert out[0].tolist() == wt and out[1].tolist() == wl and out[2].tolist() == wr and out[3].tolist() == [wm]
        mt, mr, moves = R.compact(wt, wr)
        assert moved[0].tolist() == mt and moved[1].tolist() == mr
        for c_, b in zip(cs, before):
            want = R.copied(R.copied(b, copies), [(p, q, page) for p, q in moves])
            assert all(torch.equal(x, y) for x, y in zip(c_, want))
            for x, y in zip(c_, b):
                x.copy_(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = P.fork(cs, t, n, c, ints([1, 1], dev))
    torch.cuda.current_stream().wait_stream(side)
    assert out[0].tolist() == R.fork(table, lens, refs, [1, 1], 0, page)[0]


def test_the_long_way_gives_the_same(dev, monkeypatch):
    from uwc_amd import _lib, pages as P, w4
    import w4_reference as W
    page = 16
    table, lens, refs, pages = R.state(random.Random(3), page, 4, 60, 2)
    t, n, c, parents = ints(table, dev), ints(lens, dev), ints(refs, dev), ints([0, 2, 2, -1, 1], dev)
    g = torch.Generator().manual_seed(1)
    codes, scales = (x.to(dev) for x in W.weight(64, 96, g))
    x = torch.randn((5, 96), generator=g).bfloat16().to(dev)
    bias = torch.randn(64, generator=g).bfloat16().to(dev)

    def run():
        cs = caches(2, pages, 2, 32, page, 5, dev)
        out = P.fork(cs, t, n, c, parents, room=3)
        return [*out, *P.compact(cs, out[0], out[2]), *(y for l in cs for y in l), w4.linear(x, codes, scales, bias), w4.gated(x, codes, scales)]

    short = run()
    monkeypatch.setattr(_lib, "_KV", _lib._LongWay)
    assert all(torch.equal(a, b) for a, b in zip(short, run()))


def test_two_streams_at_once(dev):
    """Calls on two streams overlap: each has its own workspace."""
    from uwc_amd import pages as P, w4
    import w4_reference as W
    page = 32
    rng = random.Random(21)
    states = [R.state(rng, page, 40, 300, 4, spare=60) for _ in range(2)]
    sets = [caches(4, s[3], 2, 64, page, i, dev) for i, s in enumerate(states)]
    parents = [[rng.randrange(-1, 40) for _ in range(60)] for _ in range(2)]
    inputs = [(ints(s[0], dev), ints(s[1], dev), ints(s[2], dev), ints(p, dev)) for s, p in zip(states, parents)]
    g = torch.Generator().manual_seed(2)
    codes, scales = (x.to(dev) for x in W.weight(512, 1024, g))
    xs = [torch.randn((m, 1024), generator=g).bfloat16().to(dev) for m in (3, 400)]
    want = [w4.linear(x, codes, scales) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((P.fork(sets[i], *inputs[i], room=5), w4.linear(xs[i], codes, scales)))
    torch.cuda.synchronize()
    for i in range(2):
        wt, wl, wr, wm, _ = R.fork(states[i][0], states[i][1], states[i][2], parents[i], 5, page)
        for (t, n, r, m), y in got[i]:
            assert t.tolist() == wt and n.tolist() == wl and r.tolist() == wr and m.tolist() == [wm] and torch.equal(y, want[i])
