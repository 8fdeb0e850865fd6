"""The layer-norm generator and the Muon optimiser together, as `train.py --type_norm LN --optimizer muon` runs them: whole train
steps against the oracle, evaluation and streamed tiles against training mode, hipGraph replay, the command line."""
import numpy as np
import pytest
import torch

from helpers import cfgs, rel_l2

pytestmark = pytest.mark.gpu
cuda = torch.device("cuda")

BASE = dict(G_ch=8, D_ch=8, z_dim=8, leak_G=0.02, n_layers_G=4, n_layers_D=3, type_norm="LN", outer_padding="replicate", base_res=4,
            num_patches_height=3, num_patches_width=3, map_dim=1, attention=False, spec_norm_D=False, padding_mode="local")


def build(a, seed=0):
    from infinite_texture_gans_amd.models.generators import ResidualPatchGenerator
    from infinite_texture_gans_amd.models.discriminators import PatchDiscriminator
    torch.manual_seed(seed)
    G = ResidualPatchGenerator(z_dim=a["z_dim"], G_ch=a["G_ch"], base_res=a["base_res"], n_layers_G=a["n_layers_G"],
                               attention=a["attention"], img_ch=3, leak=a["leak_G"], SN=False, type_norm=a["type_norm"],
                               padding_mode=a["padding_mode"], outer_padding=a["outer_padding"],
                               num_patches_h=a["num_patches_height"], num_patches_w=a["num_patches_width"])
    D = PatchDiscriminator(img_ch=3, base_ch=a["D_ch"], n_layers_D=a["n_layers_D"], kw=4, SN=a["spec_norm_D"])
    with torch.no_grad():
        for k, p in G.named_parameters():
            if ".bn" in k or k.startswith("bn."):
                p.add_(0.2 * torch.randn_like(p))
    return G.to(cuda).train(), D.to(cuda).train()


def args_of(*flags):
    from infinite_texture_gans_amd import utils as U
    args = U.prepare_parser().parse_args(list(flags))
    args.beta1 = 0.0
    return args


def inputs(a, step):
    g = torch.Generator().manual_seed(100 + step)
    z = torch.randn(2, a["z_dim"], a["num_patches_height"] * a["base_res"] + 2, a["num_patches_width"] * a["base_res"] + 2, generator=g)
    return torch.rand(4, 3, 64, 64, generator=g) * 2 - 1, z


def copies(net, dtype):
    return {k: v.detach().cpu().to(dtype) if v.is_floating_point() else v.detach().cpu().clone() for k, v in net.state_dict().items()}


@pytest.mark.parametrize("optimizer", ["muon", "adam"])
@pytest.mark.parametrize("change", [{}, {"attention": True, "n_layers_G": 4}, {"padding_mode": "zeros", "num_patches_height": 1, "num_patches_width": 1},
                                    {"spec_norm_D": True}])
def test_train_steps_match_the_oracle(change, optimizer):
    from infinite_texture_gans_amd import ops
    from infinite_texture_gans_amd.engine import Trainer
    from oracle import nets as onets, step as ostep
    from test_gpu_fullsize import _act_masks
    a = dict(BASE, **change)
    G, D = build(a)
    gcfg, dcfg = cfgs(a)
    gsd, dsd = ostep.as_leaf_params(copies(G, torch.float64)), ostep.as_leaf_params(copies(D, torch.float64))
    args = args_of("--smooth", "--optimizer", optimizer, "--muon_wd", "0.1")
    tr = Trainer(G, D, args, cuda)
    if optimizer == "muon":
        opt = [ostep.Muon([sd[k] for k in ostep.trainable(sd)], weight_decay=0.1) for sd in (dsd, gsd)]
    else:
        opt = [ostep.Adam([sd[k] for k in ostep.trainable(sd)]) for sd in (dsd, gsd)]
    for s in range(2):
        real, z = inputs(a, s)
        if a["padding_mode"] == "zeros":
            z = z[:, :, :a["base_res"], :a["base_res"]].contiguous()
        # the oracle runs on the GPU step's side of every LeakyReLU: an activation within rounding of zero may take the other
        # slope there, which moves a gradient of these small nets by some 1e-3
        ops.ACT_SINK = []
        try:
            got = [float(v) for v in tr.step(real.to(cuda), z.to(cuda), None)]
            onets.ACT_REPLAY = _act_masks(ops.ACT_SINK)
            r = ostep.train_step(gsd, dsd, gcfg, dcfg, opt[1], opt[0], real.double(), z.double(), None, smooth=True)
            assert not onets.ACT_REPLAY
        finally:
            ops.ACT_SINK = onets.ACT_REPLAY = None
        assert np.allclose(got, [r["d_loss_real"], r["d_loss_fake"], r["g_loss"]], rtol=1e-4, atol=1e-6), (s, got)
        if s == 0:
            for k, p in G.named_parameters():
                want = gsd[k].grad
                if float(want.abs().max()) < 1e-9:       # a gate at zero: no gradient behind it
                    assert float(p.grad.abs().max()) < 1e-9, k
                    continue
                assert rel_l2(p.grad.cpu(), want) < 1e-3, (k, rel_l2(p.grad.cpu(), want))
            for k, p in D.named_parameters():
                assert rel_l2(p.grad.cpu(), r["gradD"][k]) < 1e-3, k
    for net, sd in ((G, gsd), (D, dsd)):
        for k, v in net.state_dict().items():
            if k == "attention.phi.bias":      # shifts all scores of a query alike: its gradient is rounding noise, of which Adam makes +-lr
                assert float((v.cpu().double() - sd[k].detach()).abs().max()) <= 2 * 2e-4 * 2 + 1e-7
                continue
            assert rel_l2(v.cpu(), sd[k].detach()) < 2e-3, (k, rel_l2(v.cpu(), sd[k].detach()))


def test_evaluation_is_training_and_tiles_are_the_image():
    """no statistics: the same pixels in train and eval mode, whatever else is in the batch, and streamed sub-images equal the
    one-shot image"""
    from infinite_texture_gans_amd import utils as U
    G, _ = build(BASE)
    _, z = inputs(BASE, 0)
    with torch.no_grad():
        train = G(z.to(cuda))
        alone = G(z[:1].to(cuda))
        G.eval()
        assert rel_l2(G(z.to(cuda)).cpu(), train.cpu()) < 1e-6
        assert rel_l2(alone.cpu(), train[:9].cpu()) < 1e-6
        imgs = []
        for one_shot in (True, False):
            torch.manual_seed(3)
            imgs.append(U.sample_from_gen_PatchByPatch_test(G, BASE["z_dim"], BASE["base_res"], 1, num_images=1, num_patches_height=3,
                                                            num_patches_width=3, device=cuda, output_resolution_height=150,
                                                            output_resolution_width=110, one_shot=one_shot).cpu())
    assert imgs[0].shape[-2:] == (150, 110) and rel_l2(imgs[0], imgs[1]) < 1e-5


def test_graph_replays_equal_eager_steps():
    """a recorded iteration replayed four times, against the same iterations launched eagerly (two builds of one seed; D(real)'s
    weight gradients accumulate in another order under replay, and Newton-Schulz amplifies that rounding)"""
    from infinite_texture_gans_amd.engine import Trainer
    nets = [build(BASE) for _ in range(2)]
    trs = [Trainer(G, D, args_of("--smooth", "--optimizer", "muon"), cuda) for G, D in nets]
    batches = [tuple(t.to(cuda) for t in inputs(BASE, s)) for s in range(5)]
    for tr in trs:
        tr.step(*batches[0])
    trs[0].capture(*batches[0], warmup=0)
    for real, z in batches[1:]:
        a = [float(v) for v in trs[0].step_graphed(real, z)]
        b = [float(v) for v in trs[1].step(real, z)]
        assert np.allclose(a, b, rtol=1e-3, atol=1e-5), (a, b)
    for k, v in nets[0][0].state_dict().items():
        assert rel_l2(v.cpu(), nets[1][0].state_dict()[k].cpu()) < 5e-3, k


def test_flat_buffers_hold_vectors_then_matrices_and_the_ema_follows():
    from infinite_texture_gans_amd.engine import Trainer
    G, D = build(BASE)
    E, _ = build(BASE)
    before = {k: v.clone() for k, v in G.state_dict().items()}
    tr = Trainer(G, D, args_of("--optimizer", "muon", "--ema", "--ema_decay", "0.9"), cuda, netG_ema=E)
    for k, v in G.state_dict().items():
        assert torch.equal(v, before[k]), k
    assert tr.flatG.vectors == sum(p.numel() for p in G.parameters() if p.dim() < 2)
    real, z = inputs(BASE, 0)
    tr.step(real.to(cuda), z.to(cuda), None)
    for k, v in G.state_dict().items():
        want = 0.9 * before[k].double() + 0.1 * v.double()
        assert rel_l2(E.state_dict()[k].cpu(), want.cpu()) < 1e-6, k
    tr.optG.lr *= 0.5           # a decay reaches the matrices too
    p0 = tr.flatG.data.clone()
    tr.flatG.grad.copy_(torch.randn_like(p0))
    tr.optG.m.zero_()
    tr.optG.step()
    n, (r, c) = tr.flatG.vectors, tr.flatG.shapes[0]
    step = (p0 - tr.flatG.data)[n:n + r * c].view(r, c)
    s = torch.linalg.svdvals(step.cpu()) / (0.005 * max(1.0, r / c) ** 0.5)
    assert float(s.max()) < 1.3 and float(s.median()) > 0.6          # the orthogonalised update at half of 0.01


def test_unknown_choices_are_refused():
    from infinite_texture_gans_amd.engine import Trainer
    with pytest.raises(ValueError):
        build(dict(BASE, type_norm="GN"))
    G, D = build(BASE)
    with pytest.raises(ValueError):
        Trainer(G, D, args_of("--optimizer", "sgd"), cuda)


@pytest.mark.parametrize("mode", ["eager", "graph"])
def test_train_and_sample_command_lines(tmp_path, mode):
    from PIL import Image
    from infinite_texture_gans_amd import train as T, test_sample as S
    Image.fromarray(np.random.RandomState(0).randint(0, 255, (120, 160, 3), dtype=np.uint8)).save(tmp_path / "tex.jpg")
    out = tmp_path / "cp"
    T.main(["--data_path", str(tmp_path / "tex.jpg"), "--random_crop", "48", "--padding_mode", "local", "--type_norm", "LN", "--optimizer",
            "muon", "--muon_lr", "0.005", "--G_ch", "8", "--D_ch", "8", "--z_dim", "8", "--n_layers_G", "4", "--n_layers_D", "3", "--batch_size", "4",
            "--num_images", "2", "--sampling", "16", "--epochs", "2", "--saving_rate", "2", "--leak_G", "0.02", "--smooth", "--ema", "--seed", "3",
            "--decay_lr", "exp", "--launch_mode", mode, "--fname", str(out)])
    ck = torch.load(out / "2_2.pth", map_location="cpu", weights_only=False)
    keys = set(ck["netG_state_dict"])
    assert "block1.bn1.weight" in keys and "bn.bias" in keys and not any("running" in k for k in keys)
    assert all(np.isfinite(ck["Gloss"])) and all(torch.isfinite(v).all() for v in ck["netG_state_dict"].values())
    S.main(["--model_path", str(out / "2__ema.pth"), "--output_resolution_height", "100", "--output_resolution_width", "170",
            "--output_name", "gen.png"])
    assert Image.open(out / "gen.png").size == (170, 100)


def _steps(rank, world, port, out):
    """two iterations of the whole model: plain (world 0), or its patch rows sharded over ``world`` ranks"""
    import os
    import sys
    sys.path.insert(0, os.path.dirname(__file__))
    import torch.distributed as dist
    from infinite_texture_gans_amd.engine import BandTrainer, Trainer
    from infinite_texture_gans_amd.dist import BandComm
    if world > 1:
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        G, D = build(BASE)
        args = args_of("--smooth", "--optimizer", "muon")
        tr = BandTrainer(G, D, args, cuda, BandComm(rank, world)) if world else Trainer(G, D, args, cuda)
        losses = []
        for s in range(2):
            real, z = inputs(BASE, s)
            k = real.shape[0] // max(1, world)
            losses.append([float(v) for v in tr.step(real[rank * k:(rank + 1) * k].to(cuda), z.to(cuda))])
        torch.save({"losses": losses, "G": {k: v.cpu() for k, v in G.state_dict().items()},
                    "D": {k: v.cpu() for k, v in D.state_dict().items()}}, "%s.%d.%d" % (out, world, rank))
    finally:
        if world > 1:
            dist.destroy_process_group()


def test_row_sharded_steps_equal_the_plain_ones(tmp_path):
    """the generator's 3 patch rows on one rank and on two (2 + 1): no statistics are exchanged, the halo rows and gradients are.
    Other conv kernels run there: gradients differ by fp32 rounding (about 1e-5), which five Newton-Schulz steps amplify by
    3.4^5 at most - 5e-3 of an update whose singular values are 0.01 beside weights' of about 1; Adam's first steps of a vector
    are +-lr where rounding decides the sign."""
    import torch.multiprocessing as mp
    from test_gpu_model import free_port
    out = str(tmp_path / "r")
    _steps(0, 0, 0, out)
    _steps(0, 1, 0, out)
    mp.spawn(_steps, args=(2, free_port(), out), nprocs=2, join=True)
    plain = torch.load(out + ".0.0")
    runs = [[torch.load(out + ".1.0")], [torch.load(out + ".2.%d" % r) for r in range(2)]]
    for res in runs:
        for s in range(2):
            mean = np.mean([r["losses"][s] for r in res], 0)
            assert np.allclose(mean, plain["losses"][s], rtol=1e-3, atol=1e-5), (len(res), s, mean, plain["losses"][s])
        for key in ("G", "D"):
            for k, v in plain[key].items():
                got = res[0][key][k]
                assert all(torch.equal(got, r[key][k]) for r in res[1:]), k          # the replicas stay identical
                if v.dim() < 2:
                    assert float((got - v).abs().max()) <= 2 * 2e-4 * 2 + 1e-6, k
                else:
                    assert rel_l2(got, v) < 2e-3, (k, rel_l2(got, v))


# Gains, shifts and biases, whose Adam steps hide a gradient's size: the gradients themselves are compared (with 5e-3 where other
# kernels run or sums have another order: fp32 rounding is 1e-5 there, and an activation within rounding of zero that takes the other
# slope moves a gradient of these small nets by some 1e-3), and every value has to have moved by the step that its own gradient and
# second moment give.  That step is computed in 64 bits; the kernel's is off by its fp32 operations (six roundings of it at most,
# below 1e-6) and by the rounding of the value it is taken from.
def vectors_moved(flat, before, v_before, opt, t, lr=2e-4, eps=1e-8):
    n = flat.vectors
    assert n > 0
    b2 = float(torch.tensor(0.999, dtype=torch.float32))
    g, v0, p0, p1 = (x[:n].cpu().double() for x in (flat.grad, v_before, before, flat.data))
    v = b2 * v0 + (1 - b2) * g * g
    step = -lr * g / (torch.sqrt(v) / (1 - b2 ** t) ** 0.5 + eps)
    assert float(((p1 - p0) - step).abs().max()) <= 1e-5 * lr + 2 * 2.0 ** -24 * float(p0.abs().max())
    assert float((v - opt.v.cpu().double()).abs().max()) <= 1e-6 * float(v.max())
    # they have moved: in the first step every value whose gradient stands above eps by lr, later a value by sqrt(2) lr times the ratio
    # of its gradients (which may be small for one of them)
    assert float((g.abs() > 1e-6).double().mean()) > 0.9 and float((p1 - p0).abs().mean()) > 0.1 * lr


def vector_gradients(net):
    return {k: p.grad.cpu().clone() for k, p in net.named_parameters() if p.dim() < 2}


def close_gradients(got, want):
    assert set(got) == set(want)
    live = 0
    for k, g in want.items():
        if float(g.abs().max()) < 1e-9:
            assert float(got[k].abs().max()) < 1e-9, k
            continue
        live += 1
        assert rel_l2(got[k], g) < 5e-3, (k, rel_l2(got[k], g))
    assert live >= 0.9 * len(want)


def test_vectors_of_a_replayed_step():
    """the replay's gains, shifts and biases: the gradients of the same step launched eagerly, and Adam's step of them"""
    from infinite_texture_gans_amd.engine import Trainer
    nets = [build(BASE) for _ in range(2)]
    trs = [Trainer(G, D, args_of("--smooth", "--optimizer", "muon"), cuda) for G, D in nets]
    batches = [tuple(t.to(cuda) for t in inputs(BASE, s)) for s in range(3)]
    for tr in trs:
        tr.step(*batches[0])
    trs[0].capture(*batches[0], warmup=0)
    for t in (2, 3):
        before = [[(f.data.clone(), o.v.clone()) for f, o in ((tr.flatG, tr.optG), (tr.flatD, tr.optD))] for tr in trs]
        trs[0].step_graphed(*batches[t - 1])
        trs[1].step(*batches[t - 1])
        torch.cuda.synchronize()
        for tr, was in zip(trs, before):
            for flat, opt, (p0, v0) in ((tr.flatG, tr.optG, was[0]), (tr.flatD, tr.optD, was[1])):
                vectors_moved(flat, p0, v0, opt, t)
        if t == 2:                 # (later steps start from weights that differ by rounding, amplified)
            for a, b in zip(*nets):
                close_gradients(vector_gradients(a), vector_gradients(b))


def _first_step(rank, world, port, out):
    import os
    import sys
    sys.path.insert(0, os.path.dirname(__file__))
    import torch.distributed as dist
    from infinite_texture_gans_amd.engine import BandTrainer, Trainer
    from infinite_texture_gans_amd.dist import BandComm
    if world > 1:
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        G, D = build(BASE)
        args = args_of("--smooth", "--optimizer", "muon")
        tr = BandTrainer(G, D, args, cuda, BandComm(rank, world)) if world else Trainer(G, D, args, cuda)
        before = [f.data.clone() for f in (tr.flatG, tr.flatD)]
        real, z = inputs(BASE, 0)
        k = real.shape[0] // max(1, world)
        tr.step(real[rank * k:(rank + 1) * k].to(cuda), z.to(cuda))
        torch.cuda.synchronize()
        for flat, opt, p0 in ((tr.flatG, tr.optG, before[0]), (tr.flatD, tr.optD, before[1])):
            vectors_moved(flat, p0, torch.zeros_like(p0), opt, 1)
        torch.save([vector_gradients(net) for net in (G, D)], "%s.%d.%d" % (out, world, rank))
    finally:
        if world > 1:
            dist.destroy_process_group()


def test_vectors_of_row_sharded_steps(tmp_path):
    """the first step's gradients of gains, shifts and biases on one rank of patch rows and on two, against the plain step's"""
    import torch.multiprocessing as mp
    from test_gpu_model import free_port
    out = str(tmp_path / "v")
    _first_step(0, 0, 0, out)
    _first_step(0, 1, 0, out)
    mp.spawn(_first_step, args=(2, free_port(), out), nprocs=2, join=True)
    plain = torch.load(out + ".0.0")
    for name in (".1.0", ".2.0", ".2.1"):
        for got, want in zip(torch.load(out + name), plain):
            close_gradients(got, want)
