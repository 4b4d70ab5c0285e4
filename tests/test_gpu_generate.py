"""Generation over the paged 8-bit cache (uwc_amd.generate) against the same model's own forward."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(dev, mode=None, layers=2, **kw):
    transformers = pytest.importorskip("transformers")
    from uwc_amd import model as M
    cfg = dict(vocab_size=640, hidden_size=512, intermediate_size=768, num_hidden_layers=layers, num_attention_heads=8,
               num_key_value_heads=2, head_dim=64, max_position_embeddings=512, tie_word_embeddings=False)
    cfg.update(kw)
    cfg = transformers.Qwen3Config(**cfg)
    cfg._attn_implementation = "eager"
    torch.manual_seed(11)
    m = transformers.Qwen3ForCausalLM(cfg).eval().to(torch.bfloat16).to(dev)
    if mode:
        M.convert_qwen3(m, dev, mode=mode, hadamard_block=128)
    return m


def logits_of(gen, prompts, chunk):
    """Logits after every token of the prompts, the last `tail` of them as decode steps."""
    B = len(prompts)
    held = [-(-len(p) // gen.page) for p in prompts]
    pages = iter(range(sum(held)))
    table = gen._ints([[next(pages) for _ in range(n)] + [-1] * (max(held) - n) for n in held])
    out = [[] for _ in prompts]
    done = [0] * B
    while any(d < len(p) for d, p in zip(done, prompts)):
        new = [min(chunk, len(p) - d) for d, p in zip(done, prompts)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        ids = torch.tensor([t for p, d, n in zip(prompts, done, new) for t in p[d:d + n]], device=gen.dev)
        one = all(n == 1 for n in new)
        lens = [d + n for d, n in zip(done, new)]
        h = gen.forward(ids, table, gen._ints(done), gen._ints(lens), None if one else gen._ints(cu), max(new), max(lens))
        y = gen.model.lm_head(h)
        for b in range(B):
            out[b].append(y[cu[b]:cu[b + 1]])
        done = lens
    return [torch.cat(x) for x in out]


@pytest.mark.parametrize("mode", [None, "int"])
@pytest.mark.parametrize("chunk", [200, 33, 1])
def test_logits_track_the_models_own(dev, mode, chunk):
    """Keys and values rounded to 8 bits with a scale per page of 16 tokens (about 1% each, of Gaussian heads), and
    bf16 roundings between: logits within 5% of the model's own over its own cache-free forward."""
    from uwc_amd.generate import PagedGenerator
    m = build(dev, mode)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in ((70, 45) if chunk > 1 else (30, 30))]
    got = logits_of(PagedGenerator(m, pages=16, page=16), prompts, chunk)
    for p, y in zip(prompts, got):
        with torch.no_grad():
            want = m(input_ids=torch.tensor([p], device=dev), use_cache=False).logits[0].float()
        rel = ((y.float() - want).norm() / want.norm()).item()
        assert rel < 0.05, rel


def test_generate(dev):
    """Tokens are those of the logits step by step; sequences do not disturb each other; pages come back."""
    from uwc_amd.generate import PagedGenerator
    m = build(dev, "int")
    gen = PagedGenerator(m, pages=40, page=16)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in (37, 1, 64)]
    out = gen.generate(prompts, steps=20, chunk=24)
    assert [len(o) for o in out] == [20] * 3 and sorted(gen.free) == list(range(40))
    for p, o in zip(prompts, out):
        y = logits_of(gen, [p + o[:-1]], 1000)[0][len(p) - 1:].float()
        best = y.max(-1).values
        took = y.gather(1, torch.tensor(o, device=dev)[:, None])[:, 0]
        # the tokens' logits in one packed forward: near ties may turn, by the cache's rounding at most
        assert ((best - took) <= 0.05 * y.std(-1) * 4).all()
    with pytest.raises(AssertionError, match="pages are needed"):
        gen.generate([[1] * 300] * 3, steps=5)
    with pytest.raises(AssertionError, match="positions"):
        gen.generate([[1] * 510], steps=5)
    with pytest.raises(AssertionError, match="at least one"):
        gen.generate([[]], steps=5)
    assert sorted(gen.free) == list(range(40))


def test_generate_with_a_sliding_window(dev):
    """Layers whose attention slides see their window alone: logits track the model's own mask."""
    from uwc_amd.generate import PagedGenerator
    m = build(dev, None, use_sliding_window=True, sliding_window=24, max_window_layers=0, layer_types=["sliding_attention"] * 2)
    gen = PagedGenerator(m, pages=16, page=16)
    assert gen.layers[0][5] == 24
    p = torch.randint(0, 640, (100,), generator=torch.Generator().manual_seed(5)).tolist()
    y = logits_of(gen, [p], 64)[0].float()
    with torch.no_grad():
        want = m(input_ids=torch.tensor([p], device=dev), use_cache=False).logits[0].float()
    rel = ((y - want).norm() / want.norm()).item()
    assert rel < 0.05, rel
