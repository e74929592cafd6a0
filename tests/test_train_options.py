"""TuckerMoETrain's and TuckerFFNTrain's routing and 8-bit products: what needs no GPU."""
import pytest
import torch


def _layer(pkg, **kw):
    return pkg.TuckerMoETrain(64, 48, num_experts=8, r2=64, r3=64, **kw)


def test_only_a_routing_layer_has_a_bias(pkg):
    assert "balance_bias" not in _layer(pkg, fused_router=True, fp8_products=True).state_dict()
    m = _layer(pkg, routing={})
    assert m.state_dict()["balance_bias"].shape == (8,) and "balance_bias" not in dict(m.named_parameters())
    cfg = pkg.TuckerMoEConfig(kmoe_num_experts=4, kmoe_r1=4, kmoe_r2=64, kmoe_r3=64)
    f = pkg.TuckerFFNTrain(64, cfg, routing={"score": "sigmoid"}, fp8_products=True)
    assert sorted(k for k in f.state_dict() if "balance" in k) == [
        f"ffn_{n}.balance_bias" for n in ("down", "gate", "up")]
    assert all(l.fp8_products and l.routing == {"score": "sigmoid"} for l in (f.ffn_gate, f.ffn_up, f.ffn_down))
    with pytest.raises(RuntimeError, match="balance_bias"):
        pkg.TuckerFFN(64, cfg).load_state_dict(f.state_dict())


def test_the_bias_stays_float32(pkg):
    m = _layer(pkg, routing={})
    m.balance_bias.copy_(torch.linspace(-1, 1, 8) + 2.0 ** -20)
    want = m.balance_bias.clone()
    for cast in (lambda x: x.bfloat16(), lambda x: x.double(), lambda x: x.to(torch.bfloat16), lambda x: x.half()):
        cast(m)
        assert m.balance_bias.dtype == torch.float32 and torch.equal(m.balance_bias, want)
        assert m._buffers["balance_bias"] is m.balance_bias
    assert m.to("meta").balance_bias.device.type == "meta"
    assert _layer(pkg).bfloat16().U_in.dtype == torch.bfloat16


def test_update_balance(pkg):
    m = _layer(pkg, routing={})
    with pytest.raises(RuntimeError, match="follows a forward"):
        m.update_balance()
    with pytest.raises(RuntimeError, match="routing="):
        _layer(pkg, fused_router=True).update_balance()
    m.expert_counts = torch.tensor([0, 1, 2, 3, 4, 5, 6, 11])       # mean 4
    m.update_balance(0.25)
    m.update_balance(0.25)
    assert m.balance_bias.tolist() == [0.5, 0.5, 0.5, 0.5, 0.0, -0.5, -0.5, -0.5]


def test_refusals(pkg):
    with pytest.raises(ValueError, match="options are score"):
        _layer(pkg, routing={"bias": None})
    with pytest.raises(RuntimeError, match="fused_router=True or routing="):
        _layer(pkg)(torch.randn(3, 64), mask=torch.ones(3, dtype=torch.bool))
    for kw in (dict(routing={}), dict(fp8_products=True, fused_router=True)):
        with pytest.raises(RuntimeError, match="HIP"):
            _layer(pkg, **kw)(torch.randn(3, 64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_are_cast_under_autocast(pkg, monkeypatch, dtype):
    """Float32 parameters, a hidden state of either type: both products' operands are autocast's, as
    torch.matmul's in their place, and outside it they are what they are."""
    import mamba_tuckermoe_amd.latent as lat
    seen = []

    def product(x, w):
        seen.append((x.dtype, w.dtype))
        return x @ w
    monkeypatch.setattr(lat, "fp8_matmul", product)
    monkeypatch.setattr(lat.FusedLatentMoE, "apply", staticmethod(
        lambda xs, G, idx, p: torch.einsum("br,bkrs,bk->bs", xs, G[idx], p.to(xs.dtype))))
    monkeypatch.setattr(lat, "fused_router", lambda raw, k, *a: (
        *reversed(torch.softmax(raw.float(), -1).topk(k)), 0.0, 0.0, None))
    x = torch.randn(5, 64).to(dtype).requires_grad_()
    m = _layer(pkg, fused_router=True, fp8_products=True)
    with torch.autocast("cpu", torch.bfloat16):
        out, _, _ = m(x)
    out.float().square().sum().backward()
    assert seen == [(torch.bfloat16, torch.bfloat16)] * 2
    assert x.grad.dtype == dtype and all(p.grad.dtype == torch.float32 for p in m.parameters())
    if dtype == torch.float32:
        del seen[:]
        m(x)
        assert seen == [(torch.float32, torch.float32)] * 2


def test_a_layer_of_an_older_pickle(pkg, monkeypatch):
    """A whole module saved before the options existed has neither attribute: it is the layer it was."""
    import mamba_tuckermoe_amd.latent as lat
    monkeypatch.setattr(lat.FusedLatentMoE, "apply", staticmethod(
        lambda xs, G, idx, p: torch.einsum("br,bkrs,bk->bs", xs, G[idx], p)))
    m = _layer(pkg)
    x = torch.randn(5, 64)
    want, lb, z = m(x)
    for name in ("routing", "fp8_products"):
        del m.__dict__[name]
    out, lb2, z2 = m(x)
    assert torch.equal(out, want) and torch.equal(lb, lb2) and torch.equal(z, z2)
