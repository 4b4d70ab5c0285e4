"""PagedGenerator's rotation tables are the model's own for sequences of every length, or the model is refused (no GPU
needed)."""
import pytest
import torch

NAMED = dict(
    plain=None, linear=dict(rope_type="linear", factor=4.0),
    llama3=dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=128),
    yarn=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=128), dynamic=dict(rope_type="dynamic", factor=2.0),
    longrope=dict(rope_type="longrope", long_factor=[4.0] * 16, short_factor=[1.0] * 16, original_max_position_embeddings=128))


def build(name):
    transformers = pytest.importorskip("transformers")
    cfg = transformers.LlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=32, max_position_embeddings=512, rope_scaling=NAMED[name])
    if name == "longrope":
        cfg.original_max_position_embeddings = 128
    return transformers.LlamaForCausalLM(cfg).eval().to(torch.bfloat16)


def own(model, n):
    cos, sin = model.model.rotary_emb(torch.zeros(1), torch.arange(n)[None])
    return cos[0].float(), sin[0].float()


@pytest.mark.parametrize("name,positions", [("plain", 512), ("plain", 1), ("linear", 700), ("llama3", 512), ("yarn", 512),
                                            ("dynamic", 512), ("longrope", 128)])
def test_tables_are_those_of_every_length(name, positions):
    from uwc_amd.generate import PagedGenerator
    model = build(name)
    gen = PagedGenerator(model, pages=2, page=16, positions=positions)
    for n in {1, 2, positions // 2 + 1, positions} if positions > 1 else {1}:
        for a, b in zip((gen.cos, gen.sin), own(model, n)):
            assert torch.equal(a[:n], b)


@pytest.mark.parametrize("name,positions", [("dynamic", 600), ("longrope", 512), ("longrope", 129)])
def test_rotations_that_depend_on_the_length_are_refused(name, positions):
    from uwc_amd.generate import PagedGenerator
    model = build(name)
    before = own(model, 20)
    with pytest.raises(AssertionError, match="rotation at"):
        PagedGenerator(model, pages=2, page=16, positions=positions)
    assert all(torch.equal(a, b) for a, b in zip(before, own(model, 20)))  # the model is as it was
