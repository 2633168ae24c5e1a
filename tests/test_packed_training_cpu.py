"""The model options that use document masks, score caps, distance biases, scaled embeddings and routing,
together, on the CPU."""
import pytest
import torch

from oxidizr_b200.config import ConfigError, LitConfig
from oxidizr_b200.models import build_model

SEP = 3


def config(**model):
    m = {"name": "t", "hidden_size": 32, "num_layers": 2, "num_heads": 4, "kv_heads": 2, "num_experts": 8,
         "experts_per_tok": 2, "intermediate_size": 16, "vocab_size": 50, "max_seq_len": 64, "rope_theta": 10000.0,
         "dtype": "f32"}
    m.update(model)
    return LitConfig.from_dict({"model": m, "trainer": {
        "learning_rate": 1e-3, "batch_size": 2, "max_steps": 1, "num_epochs": 1, "gradient_accumulation": 1,
        "checkpoint_dir": "/tmp/oxi_packed", "log_interval": 1, "save_interval": 100, "load_balance_alpha": 0.01,
        "group_size": 4, "beta_kl": 0.04}})


OPTIONS = dict(doc_separator=SEP, attn_softcap=20.0, attn_alibi=True, embed_scale=32 ** 0.5, moe_score="sigmoid",
               moe_groups=4, moe_top_groups=2, moe_route_scale=2.5, moe_bias_rate=0.01)
LATENT = dict(kv_heads=None, kv_latent_dim=16, q_latent_dim=16, d_rope=8)


def packed(seed):
    g = torch.Generator().manual_seed(seed)
    docs = [torch.randint(4, 50, (n,), generator=g) for n in (9, 1, 14, 6)]
    row = torch.cat([torch.cat([d, torch.tensor([SEP])]) for d in docs])
    return docs, row[None]


@pytest.mark.parametrize("kind", [{}, LATENT])
def test_packed_documents_are_the_documents_alone(kind):
    """RoPE and the distance bias are relative, so a document's logits do not depend on what it is packed with."""
    model = build_model(config(**OPTIONS, **kind).model, seed=1).double()
    docs, row = packed(0)
    out = model.double().logits(row).double()
    at = 0
    for d in docs:
        alone = model.logits(torch.cat([d, torch.tensor([SEP])])[None]).double()
        # the logits are formed in f32: 32 terms of about 0.02 each, and the routing weights' f32
        assert (out[0, at:at + len(d) + 1] - alone[0]).abs().max() < 1e-4
        at += len(d) + 1


def test_without_the_separator_documents_do_see_each_other():
    docs, row = packed(0)
    model = build_model(config(**{**OPTIONS, "doc_separator": None}).model, seed=1)
    a = model.logits(row)
    other = row.clone()
    other[0, 0] = 49 if int(row[0, 0]) != 49 else 48
    assert not torch.equal(model.logits(other)[0, -5:], a[0, -5:])
    model = build_model(config(**OPTIONS).model, seed=1)
    assert torch.equal(model.logits(other)[0, -5:], model.logits(row)[0, -5:])


def test_the_selection_bias_moves_towards_balance():
    cfg = config(**OPTIONS)
    model = build_model(cfg.model, seed=2)
    _, row = packed(1)
    ids = row[:, :-1].expand(2, -1)
    loss, aux = model(ids, row[:, 1:].expand(2, -1))
    (loss + 0.01 * torch.stack(aux).mean()).backward()
    moe = model.layers[0].moe
    load = moe.route_load.clone()
    assert load.sum() == ids.numel() * 2 and (moe.route_bias == 0).all()
    assert moe.router.grad.abs().max() > 0
    model.update_route_bias()
    assert torch.equal(moe.route_bias, 0.01 * torch.sign(load.mean() - load))
    assert (moe.route_load == 0).all()
    # not in training, no load is counted
    with torch.no_grad():
        model(ids, row[:, 1:].expand(2, -1))
    assert (moe.route_load == 0).all()
    # and the bias goes into a checkpoint and comes back
    sd = model.export_ref()
    other = build_model(cfg.model, seed=3)
    other.import_ref(sd)
    assert torch.equal(other.layers[0].moe.route_bias, moe.route_bias)


def test_plain_options_change_nothing():
    """A config that spells the defaults out routes and embeds as one without them.  The spelled routing forms
    its softmax in 64 bits and rounds it once: two weights of a token apart by some steps of 2^-24, times expert
    outputs and two layers' gains below 1 here, stay under 1e-6 in logits below 1."""
    plain = build_model(config().model, seed=4)
    spelled = build_model(config(moe_score="softmax", moe_groups=1, embed_scale=1.0).model, seed=4)
    _, row = packed(2)
    assert (plain.logits(row) - spelled.logits(row)).abs().max() < 1e-6


def test_a_trainer_step(tmp_path):
    from oxidizr_b200.optim import AdamW, AdamWConfig, FlatParams
    from oxidizr_b200.trainer import Trainer
    cfg = config(**OPTIONS)
    model = build_model(cfg.model, seed=5)
    opt = AdamW(FlatParams(list(model.named_parameters()), "cpu"), AdamWConfig(lr=1e-3))
    _, row = packed(3)

    class Loader:
        def next_batch(self):
            return row[:, :-1].expand(2, -1), row[:, 1:].expand(2, -1)

        def __len__(self):
            return 1

    t = Trainer.__new__(Trainer)
    t.cfg, t.tc, t.model, t.opt, t.loader = cfg, cfg.trainer, model, opt, Loader()
    t.device, t.rank, t.world_size, t.global_step, t.cuda_graph = torch.device("cpu"), 0, 1, 0, False
    before = model.layers[1].moe.route_bias.clone()
    ce, norm = t.training_step()
    assert torch.isfinite(ce) and torch.isfinite(norm)
    assert not torch.equal(model.layers[1].moe.route_bias, before)


@pytest.mark.parametrize("bad,match", [
    (dict(doc_separator=50), "vocabulary"), (dict(doc_separator=-1), "doc_separator"), (dict(moe_bias_rate=-1.0), "moe_bias_rate"), (dict(attn_softcap=0.0), "attn_softcap"), (dict(moe_score="relu"), "moe_score"),
    (dict(moe_groups=3), "groups"), (dict(moe_groups=4, moe_top_groups=5), "groups"),
    (dict(moe_groups=8, moe_top_groups=1), "experts_per_tok"),
    (dict(doc_separator=1, mamba_layers=[0], mamba2_num_heads=8, mamba2_head_dim=8, mamba2_expand=2), "Mamba")])
def test_config_refusals(bad, match):
    with pytest.raises(ConfigError, match=match):
        config(**bad)


def _balance_rank(rank, store, out):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2)
    model = build_model(config(**OPTIONS).model, seed=6)
    _, row = packed(10 + rank)
    loss, _ = model(row[:, :-1], row[:, 1:])
    loads = [layer.moe.route_load.clone() for layer in model.layers]
    model.update_route_bias()
    torch.save((loads, [layer.moe.route_bias for layer in model.layers]), f"{out}.{rank}")
    dist.destroy_process_group()


def test_ranks_move_the_bias_by_their_common_load(tmp_path):
    import torch.multiprocessing as mp
    out = str(tmp_path / "out")
    mp.start_processes(_balance_rank, args=(str(tmp_path / "store"), out), nprocs=2, start_method="spawn")
    (l0, b0), (l1, b1) = (torch.load(f"{out}.{r}") for r in range(2))
    assert any(not torch.equal(x, y) for x, y in zip(l0, l1))
    for x, y, u, v in zip(l0, l1, b0, b1):
        total = x + y
        assert torch.equal(u, v) and torch.equal(u, 0.01 * torch.sign(total.mean() - total))


class Batches:
    def __init__(self, row, copies=2):
        self.row, self.copies = row, copies

    def next_batch(self):
        return self.row[:, :-1].expand(self.copies, -1), self.row[:, 1:].expand(self.copies, -1)


def trainer_of(cfg, model, opt, row):
    from oxidizr_b200.trainer import Trainer
    t = Trainer.__new__(Trainer)
    t.cfg, t.tc, t.model, t.opt, t.loader = cfg, cfg.trainer, model, opt, Batches(row)
    t.device, t.rank, t.world_size, t.global_step, t.cuda_graph = torch.device("cpu"), 0, 1, 0, False
    return t


def test_a_skipped_step_moves_no_bias():
    """A gradient that is not finite: the optimizer leaves the weights, and the biases stay with them."""
    from oxidizr_b200.optim import AdamW, AdamWConfig, FlatParams
    cfg = config(**OPTIONS)
    model = build_model(cfg.model, seed=5)
    opt = AdamW(FlatParams(list(model.named_parameters()), "cpu"), AdamWConfig(lr=1e-3))
    t = trainer_of(cfg, model, opt, packed(3)[1])
    t.training_step()
    assert bool(opt.updated())
    biases = [layer.moe.route_bias.clone() for layer in model.layers]
    assert any(b.any() for b in biases)
    weights = opt.flat.flat.clone()
    head = model.lm_head.detach().clone()
    with torch.no_grad():
        model.lm_head[5] = float("nan")
    _, norm = t.training_step()
    assert not torch.isfinite(norm) and not bool(opt.updated())
    for layer, b in zip(model.layers, biases):
        assert torch.equal(layer.moe.route_bias, b) and not layer.moe.route_load.any()
    with torch.no_grad():
        model.lm_head.copy_(head)
    assert torch.equal(opt.flat.flat, weights)
    t.training_step()
    assert bool(opt.updated()) and any(not torch.equal(layer.moe.route_bias, b) for layer, b in zip(model.layers, biases))


def test_selection_biases_and_checkpoints():
    """The option is turned on in a run that began without it, and off in one that had it: the first starts from zero
    biases, the second goes on routing with those it has."""
    plain, moving = config(**{**OPTIONS, "moe_bias_rate": None}), config(**OPTIONS)
    old = build_model(plain.model, seed=7)
    assert not any("selection_bias" in k for k in old.export_ref())
    new = build_model(moving.model, seed=8)
    with torch.no_grad():
        new.layers[0].moe.route_bias.fill_(9.0)
    new.import_ref(old.export_ref())
    _, row = packed(4)
    assert not new.layers[0].moe.route_bias.any()
    # (zero biases choose by s where none choose by the logits: the same order, and all else is the same)
    assert torch.equal(new.logits(row), old.logits(row))
    with torch.no_grad():
        for layer in new.layers:
            layer.moe.route_bias.copy_(torch.linspace(-1, 1, 8))
    want = new.logits(row)
    assert not torch.equal(want, old.logits(row))
    old.import_ref(new.export_ref())
    assert torch.equal(old.logits(row), want)
    loss, _ = old(row[:, :-1], row[:, 1:])
    loss.backward()
    old.update_route_bias()
    assert torch.equal(old.layers[0].moe.route_bias, torch.linspace(-1, 1, 8))  # they stay
    again = build_model(plain.model, seed=9)
    again.import_ref(old.export_ref())  # and go into the next checkpoint
    assert torch.equal(again.logits(row), want)
    new = build_model(plain.model, seed=7)
    again.import_ref(new.export_ref())
    assert again.layers[0].moe.route_bias is None


@pytest.mark.parametrize("bad,match", [
    (dict(moe_groups=0), "moe_groups"), (dict(moe_groups=-2), "moe_groups"), (dict(moe_groups=4, moe_top_groups=0), "moe_top_groups"),
    (dict(moe_top_groups=0), "moe_top_groups"), (dict(moe_route_scale=float("nan")), "moe_route_scale"),
    (dict(moe_route_scale=float("inf")), "moe_route_scale"), (dict(embed_scale=float("nan")), "embed_scale"),
    (dict(embed_scale=-float("inf")), "embed_scale")])
def test_config_refuses_what_the_first_forward_would_fail_on(bad, match):
    with pytest.raises(ConfigError, match=match):
        config(**bad)


def _expert_rank(rank, store, out):
    import torch.distributed as dist
    from oxidizr_b200.models.moe import MoE
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2)
    worst = 0.0
    for options in (OPTIONS, dict(OPTIONS, moe_score="softmax", moe_renorm=False, moe_groups=2, moe_top_groups=1)):
        cfg = config(**options).model
        sharded, whole = MoE(cfg, "cpu", torch.float64, ep_group=dist.group.WORLD), MoE(cfg, "cpu", torch.float64)
        for m in (sharded, whole):
            m.reset_parameters(0.3, torch.Generator().manual_seed(11))
            m.route_bias.copy_(torch.linspace(-0.3, 0.3, 8))
        g = torch.Generator().manual_seed(20 + rank)
        x, resid, dy = (torch.randn(1, 37, 32, generator=g, dtype=torch.float64) for _ in range(3))
        leaves = [x.clone().requires_grad_(True) for _ in range(2)]
        for m, leaf in zip((sharded, whole), leaves):
            y, aux = m(leaf, resid)
            ((y * dy).sum() + aux).backward()
            m.result = y.detach()
        for p in (whole.w_gu, whole.w_down):  # an expert's gradient is the sum over the ranks that send it tokens
            dist.all_reduce(p.grad)
        mine = slice(4 * rank, 4 * rank + 4)
        for a, b in ((sharded.result, whole.result), (leaves[0].grad, leaves[1].grad), (sharded.router.grad, whole.router.grad),
                     (sharded.w_gu.grad, whole.w_gu.grad[mine]), (sharded.w_down.grad, whole.w_down.grad[mine]),
                     (sharded.route_load, whole.route_load)):
            worst = max(worst, float((a - b).abs().max() / b.abs().max()))
        loads = [m.route_load.clone() for m in (sharded,)]
        dist.all_reduce(loads[0])
        sharded.move_route_bias(loads[0])
        biases = [torch.zeros(8) for _ in range(2)]
        dist.all_gather(biases, sharded.route_bias.float())
        assert torch.equal(*biases) and not torch.equal(biases[0], whole.route_bias.float())
    torch.save(worst, f"{out}.{rank}")
    dist.destroy_process_group()


def test_routing_options_with_experts_on_two_ranks(tmp_path):
    """Grouped, biased and scaled routing in the sharded layer and in the whole one: sums of the same terms in 64 bits but
    for the weights, which both take from the same f32 router."""
    import torch.multiprocessing as mp
    out = str(tmp_path / "out")
    mp.start_processes(_expert_rank, args=(str(tmp_path / "store"), out), nprocs=2, start_method="spawn")
    for r in range(2):
        assert torch.load(f"{out}.{r}") < 1e-6
