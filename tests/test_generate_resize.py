"""PagedGenerator.resize where memory runs out on the way: what is kept stays where the generator says it is (no GPU needed: the
pages are moved by their definition on the host)."""
import random

import pytest
import torch

import pages_reference as R

LAYERS, NOW = 3, 24


def generator(monkeypatch):
    """A generator of 24 pages with two kept prefixes on pages 20, 3, 17 and 9, 22, without a model."""
    from uwc_amd import generate

    def compact(caches, table, refs):
        t, n, moves = R.compact(table.tolist(), refs.tolist())
        page = caches[0][0].shape[2]
        for c in caches:
            for x, y in zip(c, R.copied(c, [(a, b, page) for a, b in moves])):
                x.copy_(y)
        return torch.tensor(t, dtype=torch.int32), torch.tensor(n, dtype=torch.int32)

    monkeypatch.setattr(generate.pool, "compact", compact)
    gen = object.__new__(generate.PagedGenerator)
    gen.page, gen.dev = 16, "cpu"
    g = torch.Generator().manual_seed(1)
    gen.caches = [R.cache(NOW, 2, 32, 16, g, "cpu") for _ in range(LAYERS)]
    gen.kept = [generate.Prefix([20, 3, 17], 40), generate.Prefix([9, 22], 20)]
    gen.free = [i for i in range(NOW) if i not in (20, 3, 17, 9, 22)]
    random.Random(2).shuffle(gen.free)
    return gen


def kept(gen):
    """What the prefixes hold, in their order, in every layer."""
    return [[x[p.pages].clone() for x in c] for p in gen.kept for c in gen.caches]


def check(gen, want, pages):
    """Every page is free or kept, once, in every layer's cache, and what is kept is what it was."""
    assert sorted(gen.free + [i for p in gen.kept for i in p.pages]) == list(range(pages))
    for c in gen.caches:
        assert all(x.shape[0] == pages and x.is_contiguous() for x in c)
    assert all(torch.equal(x, y) for a, b in zip(kept(gen), want) for x, y in zip(a, b))


def out_of_memory_at(monkeypatch, n):
    """The n-th copy of a tensor from now on finds no memory."""
    left = [n]

    def counted(f):
        def g(*a, **k):
            left[0] -= 1
            if left[0] == 0:
                raise torch.OutOfMemoryError("no memory")
            return f(*a, **k)
        return g

    monkeypatch.setattr(torch.Tensor, "clone", counted(torch.Tensor.clone))
    monkeypatch.setattr(torch, "cat", counted(torch.cat))


@pytest.mark.parametrize("pages", [5, 11, NOW - 1, NOW, NOW + 1, 60])
def test_resize(monkeypatch, pages):
    gen = generator(monkeypatch)
    want = kept(gen)
    gen.resize(pages)
    check(gen, want, pages)


@pytest.mark.parametrize("n", [1, 4, 5, 4 * LAYERS])
@pytest.mark.parametrize("pages", [5, 11, 60])
def test_resize_that_runs_out_of_memory(monkeypatch, pages, n):
    """At the first layer's first tensor, its last, the second layer's first, and the very last one."""
    gen = generator(monkeypatch)
    want = kept(gen)
    with monkeypatch.context() as m:
        from uwc_amd import generate
        move = generate.pool.compact

        def compact(*a):  # the pages are moved; then memory runs out
            out = move(*a)
            out_of_memory_at(m, n)
            return out

        m.setattr(generate.pool, "compact", compact)
        if pages > NOW:
            out_of_memory_at(m, n)
        with pytest.raises(torch.OutOfMemoryError):
            gen.resize(pages)
    check(gen, want, min(pages, NOW))
    gen.resize(pages)  # with memory again
    check(gen, want, pages)
