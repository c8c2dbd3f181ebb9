"""The operators together, as a model uses them: GCN_FC(norm="layer") trained with lpgnn.optim.AdamW and
evaluated in 8-bit integers, and the command line's flags for it."""
import json
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _batch(m=60, n=90, nnz=480, seed=0):
    from lpgnn import BipartiteBatch, BipartiteCSR, synth

    g = synth.uniform_lp(m, n, nnz, seed=seed)
    adj = BipartiteCSR.from_coo(g.row, g.col, g.val, g.m, g.n, device=DEV)
    dense = torch.zeros(m, n, dtype=torch.float64)
    dense[torch.as_tensor(g.row).long(), torch.as_tensor(g.col).long()] = torch.as_tensor(g.val).double()
    t = lambda a: torch.from_numpy(a).to(DEV)
    return BipartiteBatch(x_s=t(g.x_s), x_t=t(g.x_t), y_s=t(g.y_s), y_t=t(g.y_t), edge_index=adj, s_bs=g.m, t_bs=g.n), dense


def _model64(model, batch, A, feas=True):
    """The normed model in 64 bits on the CPU from its parameters (a dict name -> leaf), logits and parameters."""
    sd = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.state_dict().items()}
    left, right = batch.x_s.double().cpu(), batch.x_t.double().cpu()

    def lin(pre, agg, own):
        return agg @ sd[pre + ".lin_rel.weight"].t() + sd[pre + ".lin_rel.bias"] + own @ sd[pre + ".lin_root.weight"].t()

    def norm(x, pre):
        return torch.nn.functional.layer_norm(x, x.shape[1:], sd[pre + ".weight"], sd[pre + ".bias"], 1e-5).clamp(min=0)

    for k, pre in enumerate(["conv1"] + [f"layers.{i}" for i in range(len(model.layers))]):
        right2 = lin(pre + ".left2right", A.t() @ left, right)
        left2 = lin(pre + ".right2left", A @ right, left)
        left, right = norm(left2, f"norms.{k}.left"), norm(right2, f"norms.{k}.right")
    out = []
    for h, x, f in (("lin_left", left, batch.x_s), ("lin_right", right, batch.x_t)):
        y = torch.nn.functional.normalize(x @ sd[h + ".weight"].t() + sd[h + ".bias"], dim=-1) * 10
        f = f.double().cpu()
        y = y - 10 * torch.stack((f[:, -3] != 0, torch.zeros(len(f)).bool(), f[:, -1] != 0), 1).double()
        out.append(y)
    return out, sd


def test_forward_and_gradients():
    """fp32: an output of a hidden FC is within 2^-20 sum |a b| (its own tests' bound), here below 1e-5; each norm
    divides by a spread above 0.1 and the logits' normalisation scales by 10 / |logit| < 100: 1e-3 on logits up to 10
    and, by the same factors backwards, 1e-3 of a gradient's norm (no pre-activation of these inputs lies that near
    to a ReLU's corner)."""
    from lpgnn import GCN_FC

    batch, A = _batch()
    torch.manual_seed(3)
    model = GCN_FC(8, 8, hids=64, depth=4, dp=0.0, norm="layer").to(DEV)
    with torch.no_grad():
        for nm, p in model.named_parameters():
            if nm.startswith("norms"):
                p.add_(0.2 * torch.randn_like(p))
    lc, lv = model(batch)
    (rc, rv), sd = _model64(model, batch, A)
    assert (lc.cpu().double() - rc).abs().max() < 1e-3 and (lv.cpu().double() - rv).abs().max() < 1e-3
    gc, gv = torch.randn(lc.shape, device=DEV), torch.randn(lv.shape, device=DEV)
    torch.autograd.backward((lc, lv), (gc, gv))
    torch.autograd.backward((rc, rv), (gc.cpu().double(), gv.cpu().double()))
    for nm, p in model.named_parameters():
        want = sd[nm].grad
        assert (p.grad.cpu().double() - want).norm() <= 1e-3 * want.norm() + 1e-6, nm
    with torch.no_grad():  # the evaluation forward: the same kernels
        ec, ev = model.eval()(batch)
    assert torch.equal(ec, lc.detach()) and torch.equal(ev, lv.detach())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("opt", ["adamw", "adamw8"])
def test_training_steps(opt, dtype):
    """Steps with dropout and the clip: every parameter gets a gradient, and the step is torch.optim.AdamW's in 64
    bits from the same gradients, moments and norm (8-bit moments: from what they stand for)."""
    import adamw_ref as R
    from lpgnn import GCN_FC
    from lpgnn.train import make_optimizer, train_step

    batch, _ = _batch(seed=2)
    torch.manual_seed(1)
    model = GCN_FC(8, 8, hids=64, depth=3, norm="layer", compute_dtype=torch.float32 if dtype == "fp32" else "bf16").to(DEV)
    o, sched = make_optimizer(model, opt, 1e-3, 4, max_grad_norm=0.5)
    for k in range(3):
        before = [p.detach().double().cpu() for p in model.parameters()]
        def moments(p):
            st = o.state[p]
            if not st:
                return torch.zeros_like(p).double().cpu(), torch.zeros_like(p).double().cpu()
            if opt == "adamw":
                return st["exp_avg"].double().cpu(), st["exp_avg_sq"].double().cpu()
            dec = lambda q, s: R.decode(st[q].cpu(), st[s].cpu(), p.numel()).double().view(p.shape)
            return dec("m8", "m_scale"), dec("r8", "r_scale") ** 2
        old = [tuple(t.clone() for t in moments(p)) for p in model.parameters()]
        lr = o.param_groups[0]["lr"]
        loss = train_step(model, batch, o)
        assert torch.isfinite(loss)
        grads = [p.grad.double().cpu() for p in model.parameters()]
        norm = torch.stack([g.norm() for g in grads]).norm()
        assert abs(o.last_norm.item() - norm.item()) <= 2 ** -23 * norm.item()
        f = min(1.0, 0.5 / (norm.item() + 1e-6))
        for p, p0, g, (m, v) in zip(model.parameters(), before, grads, old):
            p64, _, v64 = R.step64(p0, g, m, v, k + 1, lr, (0.9, 0.999), 1e-8, 1e-2, f)
            # 4 roundings of p; ~20 of the update, whose parts are each below 4 lr: under 2^-20 of p and of 10 lr
            assert ((p.detach().double().cpu() - p64).abs() <= 2 ** -20 * (p64.abs() + 10 * lr)).all()
        sched.step()


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("half", [False, True])
def test_int8_evaluation_is_its_parts(normed, half):
    """quantize_int8(): each hidden layer is spmm -> linear_i8 (bits of tests/i8_ref.py) -> norm; the model is their
    composition."""
    import i8_ref as R
    from lpgnn import GCN_FC, add_knowledge, batch_to, layer_norm, quantize_i8
    from lpgnn import fc as _fc
    from lpgnn.sparse import spmm_forward

    batch, _ = _batch(seed=5)
    torch.manual_seed(2)
    model = GCN_FC(8, 8, hids=48, depth=3, norm="layer" if normed else None).to(DEV).eval()
    if half:
        model, batch = model.half(), batch_to(batch, DEV, half=True)
    with torch.no_grad():
        plain = model(batch)
        got = model.quantize_int8()(batch)
        dt = torch.float16 if half else torch.float32
        left, right = model.conv1(batch.x_s.to(dt), batch.x_t.to(dt), batch.edge_index, relu=not normed)
        act = lambda k, s, x: layer_norm(x, model.norms[k][s].weight, model.norms[k][s].bias, relu=True) if normed else x
        left, right = act(0, "left", left), act(0, "right", right)
        layer = model.layers[0]

        def direction(S, src, dst, d):
            agg = spmm_forward(S, src).cpu()
            wq, ws = quantize_i8(d.lin_rel.weight.detach(), d.lin_root.weight.detach())
            q, s, _ = R.quantize(torch.cat((agg, dst.cpu()), 1))
            return R.linear(q, s, wq.cpu(), ws.cpu(), d.lin_rel.bias.detach().float().cpu(), not normed, dt).to(DEV)

        l2 = direction(batch.edge_index.fwd, right, left, layer.right2left)
        r2 = direction(batch.edge_index.bwd, left, right, layer.left2right)
        left, right = act(1, "left", l2), act(1, "right", r2)
        left = _fc.linear(left, model.lin_left.weight, model.lin_left.bias)
        right = _fc.linear(right, model.lin_right.weight, model.lin_right.bias)
        want = add_knowledge(left, right, batch.x_s, batch.x_t)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert not torch.equal(got[0], plain[0])
        back = model.quantize_int8(False)(batch)
        assert torch.equal(back[0], plain[0]) and torch.equal(back[1], plain[1])


def test_int8_refusals():
    from lpgnn import GCN_FC

    batch, _ = _batch()
    model = GCN_FC(8, 8, hids=32, depth=3).to(DEV).eval()
    model.quantize_int8()
    with pytest.raises(RuntimeError, match="no gradient"):
        model(batch)
    with torch.no_grad():
        model(batch)
        model.layers[0].left2right.lin_rel.weight.mul_(2)
        with pytest.raises(RuntimeError, match="weights changed"):
            model(batch)
        model.quantize_int8()(batch)
        model.load_state_dict(model.state_dict())
        with pytest.raises(RuntimeError, match="weights changed"):
            model(batch)
    model.train()(batch)[0].sum().backward()  # training ignores the 8-bit weights

    from lpgnn import optim

    model.eval().quantize_int8()
    optim.AdamW(model.parameters()).step()
    with torch.no_grad(), pytest.raises(RuntimeError, match="weights changed"):
        model(batch)


def test_partitioned_graphs_are_refused():
    from lpgnn import GCN_FC
    from lpgnn.partition import lp_partition_batch
    from lpgnn import synth

    g = synth.uniform_lp(60, 90, 480, seed=0)
    b = lp_partition_batch([g.row, g.col, g.val, g.x_s, g.x_t, g.y_s, g.y_t, g.m + g.n], 1, 0, DEV)
    with pytest.raises(RuntimeError, match="whole graphs"):
        GCN_FC(8, 8, hids=16, norm="layer").to(DEV)(b)


def test_command_line_trains_and_evaluates(tmp_path):
    from lpgnn import run
    from tests.test_run import write_dataset

    data = str(tmp_path / "data")
    write_dataset(os.path.join(data, "synth", "highs-inp_tgt"), k=4)
    arch = "GCN_FC(8,8,hids=32,depth=3,norm='layer')"
    common = ["--arch", arch, "--dataset", "synth", "--data_prefix", data, "--log_prefix", str(tmp_path / "runs")]
    for opt in ("adamw", "adamw8"):
        args = run.parse_args(["train", *common, "--exp_nm", opt, "--epochs", "2", "--opt", opt, "--max_grad_norm", "1.0"])
        hist = run.run_exp(args)
        assert all(torch.isfinite(torch.tensor(hist["epoch_loss"]))) and os.path.exists(hist["checkpoint"])
        for extra in ([], ["--fp16", "1"], ["--int8", "1"], ["--int8", "1", "--fp16", "1"]):
            a = run.parse_args(["val", *common, "--load_from", hist["checkpoint"], *extra])
            model = run.make_model(a, for_eval=True)
            ds = run.LPDataset(a.dataset_processed_prefix, thresh_num=a.edge_num_thresh, device=a.dev)
            _, acc, rows = run.validation(model, ds, a)
            assert 0 <= acc <= 1 and len(rows) == len(ds) and json.dumps(rows)


def test_int8_refuses_gradients_of_hidden_layers_behind_frozen_ones():
    """conv1 frozen, the hidden layers not: a loss would leave them without a gradient.  Frozen too, the heads train."""
    from lpgnn import GCN_FC

    batch, _ = _batch()
    model = GCN_FC(8, 8, hids=32, depth=3).to(DEV).eval()
    model.conv1.requires_grad_(False)
    model.quantize_int8()
    with pytest.raises(RuntimeError, match="no gradient"):
        model(batch)
    model.layers.requires_grad_(False)
    model(batch)[0].square().sum().backward()
    assert model.lin_left.weight.grad is not None and model.conv1.left2right.lin_rel.weight.grad is None


def test_the_shallowest_model():
    """depth=1 is conv1 and the heads, as depth=2."""
    from lpgnn import GCN_FC

    batch, A = _batch()
    torch.manual_seed(4)
    model = GCN_FC(8, 8, hids=32, depth=1, norm="layer").to(DEV)
    lc, lv = model(batch)
    (rc, rv), _ = _model64(model, batch, A)  # (bound: test_forward_and_gradients)
    assert (lc.cpu().double() - rc).abs().max() < 1e-3 and (lv.cpu().double() - rv).abs().max() < 1e-3


@pytest.mark.parametrize("seed,hids", [(5, 64), (6, 128)])
def test_int8_evaluation_stays_near_full_precision(seed, hids):
    """How far 8 bits move the model from its definition in 64 bits.  A code is off by at most half a unit, so a hidden
    pre-activation by d = sum_k +- (s/2) |w_k| +- (ws/2) |x_k|: certainly below the sum of magnitudes, and, the roundings
    being unrelated, below t = 6.5 root sum squares (Hoeffding: 1.3e-9 each; fp32's own 1e-5 is far below t / 6).  Heads
    and logits follow: the roundings of a row through W_head, a hidden number that t can push across the ReLU's corner
    counted in full; 10 h / |h| moves by at most 20 |dh| / |h|.  Where the two best logits are further apart than twice
    that the answer is the same one."""
    import i8_ref as R
    from lpgnn import GCN_FC
    from lpgnn.conv import two_direction_i8

    batch, A = _batch(seed=seed)
    torch.manual_seed(2)
    model = GCN_FC(8, 8, hids=hids, depth=3).to(DEV).eval()
    with torch.no_grad():
        got = model.quantize_int8()(batch)
        l1, r1 = model.conv1(batch.x_s, batch.x_t, batch.edge_index, relu=True)
        hidden = two_direction_i8(l1, r1, batch.edge_index, model._int8[0], False)
    sd = {k: v.double().cpu() for k, v in model.state_dict().items()}
    left, right = batch.x_s.double().cpu(), batch.x_t.double().cpu()

    def parts(pre, agg, own):
        return torch.cat((agg, own), 1), torch.cat((sd[pre + ".lin_rel.weight"], sd[pre + ".lin_root.weight"]), 1), \
            sd[pre + ".lin_rel.bias"]

    def lin(x, W, b):
        return x @ W.t() + b

    l1, r1 = (lin(*parts("conv1.right2left", A @ right, left)).clamp(min=0),
              lin(*parts("conv1.left2right", A.t() @ left, right)).clamp(min=0))
    sides = (("layers.0.right2left", A @ r1, l1, "lin_left", left, hidden[0], got[0]),
             ("layers.0.left2right", A.t() @ l1, r1, "lin_right", right, hidden[1], got[1]))
    for pre, agg, own, head, feas, z8, logits in sides:
        x, W, b = parts(pre, agg, own)
        s, ws = (R.quantize(t.float())[1].double()[:, None] / 2 for t in (x, W))
        xq = x.abs() + s  # (no less than what the codes stand for)
        z = lin(x, W, b)
        dz = (z8.double().cpu() - z).abs()
        assert (dz <= s * W.abs().sum(1) + xq.sum(1, keepdim=True) * ws.t() + 1e-5).all()
        t = 6.5 * (s.square() * W.square().sum(1) + xq.square().sum(1, keepdim=True) * ws.square().t()).sqrt()
        assert (dz <= t).all() and t.median() < 0.2 * z.abs().median()
        Wh = sd[head + ".weight"]
        on, corner = (z > t).double(), (z.abs() <= t).double()
        h = z.clamp(min=0) @ Wh.t() + sd[head + ".bias"]
        dh = torch.stack([6.5 * (((on * w) @ W).square().sum(1) * s[:, 0].square()
                                 + (on * w).square() @ ws[:, 0].square() * xq.square().sum(1)).sqrt()
                          + (corner * t) @ w.abs() for w in Wh], 1)
        bound = 20 * dh.norm(dim=1) / h.norm(dim=1)
        y = 10 * h / h.norm(dim=1, keepdim=True)
        y = y - 10 * torch.stack((feas[:, -3] != 0, torch.zeros(len(feas)).bool(), feas[:, -1] != 0), 1).double()
        assert ((logits.double().cpu() - y).abs() <= bound[:, None] + 1e-3).all()
        best = y.topk(2, 1).values
        sure = best[:, 0] - best[:, 1] > 2 * bound
        assert sure.any() and torch.equal(logits.cpu().argmax(1)[sure], y.argmax(1)[sure])
