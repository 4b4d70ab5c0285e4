"""model.convert_4bit refuses a model as a whole: what it cannot convert anywhere is found before anything is replaced (no GPU needed)."""
import pytest
import torch

from test_gpu_generate import build


def spoiled(name, value):
    def f(m):
        m.get_submodule(name).weight.data[3, 5] = value
        return m
    return f


def biased(m):
    m.model.layers[1].mlp.up_proj.bias = torch.nn.Parameter(torch.zeros(768, dtype=torch.bfloat16))
    return m


@pytest.mark.parametrize("kw,change,msg", [
    (dict(intermediate_size=100), None, r"layers.0.*down_proj.*multiple of 32"),
    (dict(num_attention_heads=3, head_dim=24, num_key_value_heads=1), None, r"layers.0.*o_proj.*multiple of 32"),
    ({}, lambda m: m.float(), "float32"),
    ({}, lambda m: (m.model.layers[1].self_attn.o_proj.float(), m)[1], r"layers.1.*o_proj.*float32"),
    ({}, spoiled("model.layers.1.mlp.down_proj", float("inf")), r"layers.1.*down_proj.*finite"),
    ({}, spoiled("model.layers.1.self_attn.v_proj", float("nan")), r"layers.1.*v_proj.*finite"),
    ({}, spoiled("lm_head", float("-inf")), "lm_head.*finite"),
    ({}, biased, "no bias"),
])
def test_nothing_is_replaced_in_a_model_that_is_refused(kw, change, msg):
    from uwc_amd import model as M
    m = build("cpu", **kw)
    m = change(m) if change else m
    before = [(n, id(x)) for n, x in m.named_modules()], [(n, id(x), x.clone()) for n, x in m.named_parameters()]
    with pytest.raises(AssertionError, match=msg):
        M.convert_4bit(m, "cpu", lm_head=True)
    assert [(n, id(x)) for n, x in m.named_modules()] == before[0]
    for (n, x), (n0, i, x0) in zip(m.named_parameters(), before[1]):
        assert n == n0 and id(x) == i and torch.equal(x.nan_to_num(), x0.nan_to_num())


def test_what_is_left_alone_need_not_be_convertible():
    from uwc_amd import model as M
    m = spoiled("lm_head", float("inf"))(build("cpu"))
    assert len(M.convert_4bit(m, "cpu")) == 2 * 3 and isinstance(m.lm_head, torch.nn.Linear)
    m = build("cpu")
    assert len(M.convert_4bit(m.half().model, "cpu", lm_head=True)) == 2 * 3  # the bare model
