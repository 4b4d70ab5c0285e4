"""Models with 4-bit weights and beam search over shared pages: the new operators together, as generation uses them."""
import pytest
import torch

from test_gpu_generate import build, logits_of
from test_gpu_generate_models import llama

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def rounded(m):
    """The model with every 4-bit weight's values in its own type: what convert_4bit stands for."""
    from uwc_amd import w4
    for layer in m.model.layers:
        for lin in (layer.self_attn.q_proj, layer.self_attn.k_proj, layer.self_attn.v_proj, layer.self_attn.o_proj,
                    layer.mlp.gate_proj, layer.mlp.up_proj, layer.mlp.down_proj):
            lin.weight.data = w4.values(*w4.quantize(lin.weight.data), dtype=lin.weight.dtype)
    m.lm_head.weight.data = w4.values(*w4.quantize(m.lm_head.weight.data), dtype=m.lm_head.weight.dtype)
    return m


@pytest.mark.parametrize("make", [lambda dev: build(dev), lambda dev: llama(dev, HF), lambda dev: llama(dev, BF, attention_bias=True)])
def test_models_with_4_bit_weights_track_the_rounded_model(dev, make):
    """Weights of a few bits are exact in either model's type: its own forward over the same values differs by roundings between
    alone (16-bit activations through two layers, well under 2%)."""
    from uwc_amd import model as M
    want = rounded(make(dev))
    m = make(dev)
    mods = M.convert_4bit(m, dev, lm_head=True)
    assert len(mods) == 2 * 3 + 1 and not any(isinstance(x, torch.nn.Linear) for x in m.modules())
    ids = torch.randint(0, 640, (2, 50), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        a, b = (x(input_ids=ids, use_cache=False).logits.float() for x in (m, want))
    assert (a - b).norm() / b.norm() < 0.02


@pytest.mark.parametrize("chunk", [200, 33, 1])
def test_generation_with_4_bit_weights(dev, chunk):
    from uwc_amd import model as M
    from uwc_amd.generate import PagedGenerator
    want = rounded(build(dev))
    m = build(dev)
    M.convert_4bit(m, dev, lm_head=True)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in ((70, 45) if chunk > 1 else (20, 20))]
    for p, y in zip(prompts, logits_of(PagedGenerator(m, pages=16, page=16), prompts, chunk)):
        with torch.no_grad():
            ref = want(input_ids=torch.tensor([p], device=dev), use_cache=False).logits[0].float()
        assert ((y.float() - ref).norm() / ref.norm()).item() < 0.05  # 8-bit keys and values, as for other linears


def logp_of(gen, prompt, tokens):
    y = logits_of(gen, [prompt + tokens[:-1]], 1000)[0][len(prompt) - 1:].float()
    p = torch.log_softmax(y, -1).gather(1, torch.tensor(tokens, device=gen.dev)[:, None])
    return p.sum().item(), y.std(-1).mean().item()


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("prefix", [0, 9, 32, 45])
def test_beams(dev, four_bit, prefix):
    """Each beam's score is what its tokens get in one forward of their own, up to the 8-bit cache's rounding (0.05 of the logits' spread a
    step, four steps' worth of slack as in greedy generation); beams differ, come best first, and the pool is as it was."""
    from uwc_amd import model as M
    from uwc_amd.generate import PagedGenerator
    m = build(dev)
    if four_bit:
        M.convert_4bit(m, dev)
    gen = PagedGenerator(m, pages=120, page=16)
    g = torch.Generator().manual_seed(3 + prefix)
    head = torch.randint(0, 640, (prefix,), generator=g).tolist()
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in (37, 1, 16)]
    kept = gen.keep(head, chunk=20) if prefix else None
    before = [tuple(x[kept.pages].clone() for x in c) for c in gen.caches] if prefix else []
    free = sorted(gen.free)
    out = gen.beam(prompts, steps=21, beams=4, prefix=kept, chunk=24)
    assert sorted(gen.free) == free and len(free) == 120 - (-(-prefix // 16))
    for c, b in zip(gen.caches, before):  # what is kept is not written
        n = prefix - (len(kept.pages) - 1) * 16
        last = kept.pages[-1]
        assert all(torch.equal(x[kept.pages[:-1]], y[:-1]) for x, y in zip(c, b))
        assert torch.equal(c[0][last, :, :n], b[0][-1, :, :n]) and torch.equal(c[1][last, :, :, :n], b[1][-1, :, :, :n])
        assert torch.equal(c[2][last], b[2][-1]) and torch.equal(c[3][last], b[3][-1])
    for p, beams in zip(prompts, out):
        scores = [s for _, s in beams]
        assert len(beams) == 4 and scores == sorted(scores, reverse=True) and len({tuple(t) for t, _ in beams}) == 4
        for t, s in beams:
            want, spread = logp_of(gen, head + p, t)
            assert len(t) == 21 and abs(s - want) <= 0.05 * spread * 4 * 21 ** 0.5


def test_one_beam_is_greedy(dev):
    from uwc_amd.generate import PagedGenerator
    gen = PagedGenerator(build(dev), pages=60, page=16)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in (40, 40, 40)]
    assert [b[0][0] for b in gen.beam(prompts, steps=20, beams=1)] == gen.generate(prompts, steps=20)


def test_kept_prefixes_survive_a_smaller_and_a_larger_pool(dev):
    from uwc_amd.generate import PagedGenerator
    gen = PagedGenerator(build(dev), pages=90, page=16)
    g = torch.Generator().manual_seed(5)
    a, b, c = ([gen.keep(torch.randint(0, 640, (n,), generator=g).tolist()) for n in (100, 30, 77)])
    prompt = [torch.randint(0, 640, (11,), generator=g).tolist()]
    want = [gen.beam(prompt, steps=5, beams=2, prefix=p) for p in (a, c)]
    gen.forget(b)
    gen.resize(40)
    assert sorted(a.pages + c.pages + gen.free) == list(range(40)) and sorted(a.pages + c.pages) == list(range(12))
    assert [gen.beam(prompt, steps=5, beams=2, prefix=p) for p in (a, c)] == want
    gen.resize(64)
    assert sorted(a.pages + c.pages + gen.free) == list(range(64))
    assert [gen.beam(prompt, steps=5, beams=2, prefix=p) for p in (a, c)] == want
    for bad, msg in ((lambda: gen.resize(11), "in use"), (lambda: gen.forget(b), "not kept"), (lambda: gen.beam(prompt, 5, 2, prefix=b), "not kept"),
                     (lambda: gen.beam(prompt, 5, 0), "beams"), (lambda: gen.beam(prompt, 5, 641), "beams"), (lambda: gen.beam([[]], 5, 2), "at least one"),
                     (lambda: gen.beam(prompt * 30, 60, 8), "pages are needed"), (lambda: gen.beam(prompt, 500, 2, prefix=a), "positions"),
                     (lambda: gen.keep([]), "at least one"), (lambda: gen.keep([1] * 1000), "positions")):
        with pytest.raises(AssertionError, match=msg):
            bad()
    gen.forget(a), gen.forget(c)
    gen.resize(3)
    assert gen.free == [0, 1, 2]


def test_4_bit_modules_refuse(dev):
    from uwc_amd import model as M
    m = llama(dev, BF, hidden_act="gelu")
    with pytest.raises(AssertionError, match="silu"):
        M.convert_4bit(m, dev)
    assert isinstance(m.model.layers[0].self_attn.q_proj, torch.nn.Linear)  # nothing was replaced
    m = llama(dev, BF, mlp_bias=True)
    with pytest.raises(AssertionError, match="no bias"):
        M.convert_4bit(m, dev)
