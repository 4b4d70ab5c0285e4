"""A pool that cannot be made smaller for want of memory: what is kept in it is still there."""
import pytest
import torch

from test_gpu_generate import build

pytestmark = pytest.mark.gpu


def test_a_kept_prefix_survives_a_resize_that_fails(dev, monkeypatch):
    from uwc_amd.generate import PagedGenerator
    gen = PagedGenerator(build(dev), pages=60, page=16)
    g = torch.Generator().manual_seed(6)
    gone, kept = (gen.keep(torch.randint(0, 640, (n,), generator=g).tolist()) for n in (100, 77))
    prompt = [torch.randint(0, 640, (11,), generator=g).tolist()]
    want = gen.beam(prompt, steps=5, beams=2, prefix=kept)
    gen.forget(gone)
    clone, calls = torch.Tensor.clone, []

    def second_layer_has_no_memory(x, *a, **k):
        calls.append(1)
        if len(calls) == 6:
            raise torch.OutOfMemoryError("no memory")
        return clone(x, *a, **k)

    with monkeypatch.context() as m, pytest.raises(torch.OutOfMemoryError):
        m.setattr(torch.Tensor, "clone", second_layer_has_no_memory)
        gen.resize(30)
    assert sorted(kept.pages + gen.free) == list(range(30))
    gen.generate(prompt * 20, steps=5)  # writes every page that it takes for free
    assert gen.beam(prompt, steps=5, beams=2, prefix=kept) == want
    gen.resize(20)
    assert gen.beam(prompt, steps=5, beams=2, prefix=kept) == want
