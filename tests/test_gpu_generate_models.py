"""Generation over the paged 8-bit cache (uwc_amd.generate) for Llama models, heads of 128, float16 and mined linears."""
import numpy as np
import pytest
import torch

from test_gpu_generate import logits_of

pytestmark = pytest.mark.gpu


def llama(dev, dtype, mode=None, **kw):
    transformers = pytest.importorskip("transformers")
    from uwc_amd import model as M
    cfg = dict(vocab_size=640, hidden_size=512, intermediate_size=768, num_hidden_layers=2, num_attention_heads=8,
               num_key_value_heads=2, head_dim=64, max_position_embeddings=512, tie_word_embeddings=False)
    cfg.update(kw)
    cfg = transformers.LlamaConfig(**cfg)
    cfg._attn_implementation = "eager"
    torch.manual_seed(17)
    m = transformers.LlamaForCausalLM(cfg).eval().to(dtype).to(dev)
    if mode:
        M.convert_qwen3(m, dev, mode=mode, hadamard_block=128)
    return m


SCALED = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64)


@pytest.mark.parametrize("dtype,mode,kw", [
    (torch.bfloat16, None, {}), (torch.float16, None, dict(num_key_value_heads=8)), (torch.bfloat16, "int", dict(head_dim=128)),
    (torch.bfloat16, None, dict(rope_scaling=SCALED)), (torch.bfloat16, None, dict(attention_bias=True, head_dim=32)),
])
@pytest.mark.parametrize("chunk", [200, 33])
def test_llama_logits_track_the_models_own(dev, dtype, mode, kw, chunk):
    """As for the other models: 8-bit keys and values (about 1% each) and 16-bit roundings, logits within 5%."""
    from uwc_amd.generate import PagedGenerator
    m = llama(dev, dtype, mode, **kw)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 640, (n,), generator=g).tolist() for n in (70, 45)]
    gen = PagedGenerator(m, pages=16, page=16)
    for p, y in zip(prompts, logits_of(gen, prompts, chunk)):
        with torch.no_grad():
            want = m(input_ids=torch.tensor([p], device=dev), use_cache=False).logits[0].float()
        rel = ((y.float() - want).norm() / want.norm()).item()
        assert rel < 0.05, rel


def test_mined_linears_generate_what_integer_ones_do(dev):
    """Mined linears are exact: the same logits, bit for bit, and the same tokens."""
    from uwc_amd import model as M
    from uwc_amd.generate import PagedGenerator
    got = []
    for mode in ("int", "mined"):
        m = llama(dev, torch.bfloat16, vocab_size=2048, hidden_size=2048, intermediate_size=2048, num_attention_heads=16,
                  num_key_value_heads=8, head_dim=128, max_position_embeddings=256)
        mls = M.convert_qwen3(m, dev, mode=mode, hadamard_block=512)
        for ml in mls:
            ml.setup_block(lambda k: bytes(range(32)), lambda k: np.full(8, 0xFFFFFFFF, np.uint32))
        gen = PagedGenerator(m, pages=16, page=16)
        prompts = [torch.randint(0, 2048, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (40, 7)]
        got.append((logits_of(gen, prompts, 24), gen.generate(prompts, steps=6, chunk=24)))
        assert mode == "int" or sum(ml.hashed_macs for ml in mls) > 0
    assert got[0][1] == got[1][1]
    for a, b in zip(got[0][0], got[1][0]):
        assert torch.equal(a, b)
