"""Fused linears under torch.inference_mode, whose tensors count no versions (no GPU needed: the fused product is torch's)."""
import pytest
import torch


class Fused(torch.nn.Module):
    splits, calls = [3, 2, 4], 0

    def forward(self, x):
        self.calls += 1
        return x @ torch.arange(45.0).view(5, 9)


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 0, 1), (1, 1, 1)])
def test_parts_of_inference_tensors(order):
    from uwc_amd import model as M
    ml = Fused()
    parts = [M._Part(M._SharedOutput(ml), i) for i in range(3)]
    shared = parts[0].shared
    for p in parts:
        p.shared = shared
    with torch.inference_mode():
        x = torch.randn(2, 5)
        want = ml(x).split(ml.splits, -1)
        for i in order:
            assert torch.equal(parts[i](x), want[i])
        x += 1  # nothing of before is handed out
        want = ml(x).split(ml.splits, -1)
        for i in order:
            assert torch.equal(parts[i](x), want[i])
        assert torch.equal(parts[0](x), want[0])
        x.zero_()
        assert not parts[1](x).any()
    x = torch.randn(2, 5)  # outside it one product serves all three, as ever
    ml.calls = 0
    for i in range(3):
        parts[i](x)
    assert ml.calls == 1


def test_a_part_is_computed_alone_where_the_linear_can():
    from uwc_amd import model as M

    class Alone(Fused):
        def part(self, x, index):
            return (x @ torch.arange(45.0).view(5, 9)).split(self.splits, -1)[index]

    ml = Alone()
    shared = M._SharedOutput(ml)
    with torch.inference_mode():
        x = torch.randn(2, 5)
        want = ml(x).split(ml.splits, -1)
        ml.calls = 0
        assert all(torch.equal(M._Part(shared, i)(x), want[i]) for i in range(3)) and ml.calls == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
def test_a_4_bit_model_in_inference_mode(dev, bias):
    """The same weights by parts instead of fused: the sums' order may differ (fp32, far below a step of bf16), so roundings of 16-bit
    activations through two layers, under 2%."""
    from test_gpu_generate_models import llama
    from uwc_amd import model as M
    m = llama(dev, torch.bfloat16, attention_bias=bias)
    if bias:
        for layer in m.model.layers:
            for p in (layer.self_attn.q_proj, layer.self_attn.k_proj, layer.self_attn.v_proj):
                p.bias.data.normal_()
    M.convert_4bit(m, dev, lm_head=True)
    ids = torch.randint(0, 640, (2, 50), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        want = m(input_ids=ids, use_cache=False).logits.float()
    with torch.inference_mode():
        got = m(input_ids=ids, use_cache=False).logits.float()
        x = torch.randn((7, 512), device=dev, dtype=torch.bfloat16)
        att = m.model.layers[0].self_attn
        parts = [p(x) for p in (att.q_proj, att.k_proj, att.v_proj)]
        whole = att.q_proj.ml(x).split(att.q_proj.ml.splits, -1)
    assert (got - want).norm() / want.norm() < 0.02
    assert all((a.float() - b.float()).norm() / b.float().norm() < 2.0 ** -8 for a, b in zip(parts, whole))


@pytest.mark.gpu
def test_an_integer_model_in_inference_mode(dev):
    """Integer linears are exact: the same bits."""
    from test_gpu_generate import build
    m = build(dev, "int")
    ids = torch.randint(0, 640, (2, 50), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        want = m(input_ids=ids, use_cache=False).logits
    with torch.inference_mode():
        assert torch.equal(m(input_ids=ids, use_cache=False).logits, want)
