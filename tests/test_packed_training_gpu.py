"""A training step with document masks, capped scores, a distance bias, scaled embeddings and grouped sigmoid
routing together, through the kernels."""
import pytest
import torch

from oxidizr_b200.config import LitConfig
from oxidizr_b200.models import build_model

pytestmark = pytest.mark.gpu
SEP = 7


def config(**model):
    m = {"name": "t", "hidden_size": 256, "num_layers": 2, "num_heads": 4, "kv_heads": 2, "num_experts": 16,
         "experts_per_tok": 4, "intermediate_size": 128, "vocab_size": 500, "max_seq_len": 512, "rope_theta": 10000.0,
         "dtype": "bf16", "doc_separator": SEP, "attn_softcap": 30.0, "attn_alibi": True, "embed_scale": 16.0,
         "moe_score": "sigmoid", "moe_groups": 4, "moe_top_groups": 2, "moe_route_scale": 2.5, "moe_bias_rate": 1e-3}
    m.update(model)
    return LitConfig.from_dict({"model": m, "trainer": {
        "learning_rate": 1e-3, "batch_size": 2, "max_steps": 1, "num_epochs": 1, "gradient_accumulation": 1,
        "checkpoint_dir": "/tmp/oxi_packed", "log_interval": 1, "save_interval": 100, "load_balance_alpha": 0.01,
        "group_size": 4, "beta_kl": 0.04}}).model


LATENT = dict(kv_heads=None, kv_latent_dim=128, q_latent_dim=128, d_rope=32)


def batch(seed, S=300):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(8, 500, (2, S + 1), generator=g)
    for b, cuts in enumerate(((40, 41, 170, 260), (128, 255))):
        for c in cuts:
            ids[b, c] = SEP
    return ids.cuda()


def step(model, ids):
    for p in model.parameters():
        p.grad = None
    loss, aux = model(ids[:, :-1], ids[:, 1:])
    total = loss.float() + 0.01 * torch.stack([a.float() for a in aux]).mean()
    total.backward()
    return total.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("kind", [{}, LATENT])
def test_documents_do_not_see_each_other(kind):
    """What one document holds changes no bit of another's logits."""
    model = build_model(config(**kind), device="cuda", seed=1)
    ids = batch(0)[:, :-1]
    other = ids.clone()
    other[0, 50:160] = other[0, 50:160] % 400 + 50
    a, b = model.logits(ids), model.logits(other)
    assert torch.equal(a[0, :41], b[0, :41]) and torch.equal(a[0, 171:], b[0, 171:]) and torch.equal(a[1], b[1])
    assert not torch.equal(a[0, 60:171], b[0, 60:171])
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", [{}, LATENT])
def test_step_is_near_the_stated_math(kind):
    """Loss and gradients beside the same weights in f32 on the CPU.  A bf16 step rounds every activation and
    gradient by up to 2^-8 about twenty times in a row over two layers: 20 x 2^-8 of a gradient's norm is 8 %; and a
    token whose choice of experts a rounding changes moves an expert's gradient by its share (4 of 600 tokens)."""
    cfg = config(**kind)
    model = build_model(cfg, device="cuda", seed=2)
    wide = build_model(config(dtype="f32", **kind), seed=2)
    wide.import_ref({k: v.float().cpu() for k, v in model.export_ref().items()})
    ids = batch(1)
    loss, grads = step(model, ids)
    want, ref = step(wide, ids.cpu())
    assert abs(loss.item() - want.item()) < 2 ** -8 * want.item()
    for n, g in grads.items():
        r = ref[n].cuda()
        off = (g.float() - r).norm() / r.norm().clamp_min(1e-6)
        assert off < 0.16, (n, off.item())
    from oxidizr_b200.ops._C import check_status
    torch.cuda.synchronize()
    check_status("cuda")


def test_captured_step():
    """The whole training step in a graph, with other documents at each replay."""
    from oxidizr_b200.optim import AdamW, AdamWConfig, FlatParams

    def make():
        m = build_model(config(), device="cuda", seed=3)
        return m, AdamW(FlatParams(list(m.named_parameters()), "cuda"), AdamWConfig(lr=1e-3))

    def train(m, o, ids):
        loss, aux = m(ids[:, :-1], ids[:, 1:])
        (loss.float() + 0.01 * torch.stack([a.float() for a in aux]).mean()).backward()
        n = o.step()
        m.update_route_bias()
        return loss.detach(), n

    eager, eo = make()
    batches = [batch(s) for s in range(4)]
    for b in batches:
        want = train(eager, eo, b)[0].clone()
    model, opt = make()
    static = batches[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for b in batches[:2]:
            static.copy_(b)
            train(model, opt, static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = train(model, opt, static)[0]
    for b in batches[2:]:
        static.copy_(b)
        graph.replay()
    torch.cuda.synchronize()
    # other kernels of the step add gradients with atomics: f32 rounding, grown over four steps
    assert abs(loss.item() - want.item()) < 1e-2 * want.item()
    # (a near tie in the choice may fall the other way after those: the biases agree but for single steps of it)
    a, b = eager.layers[0].moe.route_bias, model.layers[0].moe.route_bias
    assert (a != 0).any() and (a - b).abs().max() <= 4 * 2 * 1e-3


@pytest.mark.parametrize("captured", [False, True])
def test_a_skipped_step_moves_no_bias(captured):
    """A gradient norm that is not finite skips the update on the device; the selection biases stay too, with no host sync."""
    from oxidizr_b200.optim import AdamW, AdamWConfig, FlatParams
    model = build_model(config(), device="cuda", seed=3)
    opt = AdamW(FlatParams(list(model.named_parameters()), "cuda"), AdamWConfig(lr=1e-3))
    ids = batch(5)

    def train():
        loss, aux = model(ids[:, :-1], ids[:, 1:])
        (loss.float() + 0.01 * torch.stack([a.float() for a in aux]).mean()).backward()
        opt.step()
        model.update_route_bias(opt.updated())

    run = train
    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            train()
            train()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            train()
        run = graph.replay
    run()
    torch.cuda.synchronize()
    assert bool(opt.updated())
    biases = [layer.moe.route_bias.clone() for layer in model.layers]
    keep = model.norm.weight.detach().clone()
    with torch.no_grad():
        model.norm.weight.fill_(float("nan"))
    run()
    torch.cuda.synchronize()
    assert not bool(opt.updated())
    for layer, b in zip(model.layers, biases):
        assert b.any() and torch.equal(layer.moe.route_bias, b) and not layer.moe.route_load.any()
    with torch.no_grad():
        model.norm.weight.copy_(keep)
    run()
    torch.cuda.synchronize()
    assert bool(opt.updated())
    assert any(not torch.equal(layer.moe.route_bias, b) for layer, b in zip(model.layers, biases))


@pytest.mark.parametrize("kind", [{}, LATENT])
def test_gradients_outside_the_experts_are_near_the_stated_math(kind):
    """The bound that twenty roundings to bf16 in a row give, 20 x 2^-8 of a gradient's norm: of the parameters that every
    token passes through, whose gradients a changed choice of experts (4 of 600 tokens) reaches through a residual."""
    model = build_model(config(**kind), device="cuda", seed=2)
    wide = build_model(config(dtype="f32", **kind), seed=2)
    wide.import_ref({k: v.float().cpu() for k, v in model.export_ref().items()})
    ids = batch(1)
    grads, ref = step(model, ids)[1], step(wide, ids.cpu())[1]
    seen = 0
    for n, g in grads.items():
        if ".moe." not in n:
            r = ref[n].cuda()
            assert (g.float() - r).norm() <= 20 * 2 ** -8 * r.norm(), (n, ((g.float() - r).norm() / r.norm()).item())
            seen += 1
    assert seen >= 8
    torch.cuda.synchronize()
