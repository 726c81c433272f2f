"""Encoders on the row-norm kernels (norm_type "rms"; "ln" under KernelOptions.fused_row_norm) and trained by optim.Muon, against
the same networks with both replaced by their formulas in 64 bits."""
import random

import pytest
import torch

from test_muon import update64
from test_rownorm import normed

BASE = dict(activation="gelu", first_stride=1, global_pool="sum", bias=True, bn_momentum=0.1, dropout=0.0, drop_path=0.3)


def plain_act(u, act):
    return {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[act or "none"](u)


def plain_row_norm(x, weight=None, bias=None, eps=1e-6, kind="layer", act=None):
    n = normed(x.double(), kind, eps) * weight.double()
    return plain_act(n if bias is None else n + bias.double(), act).to(x.dtype)


def plain_join(z, r, weight=None, bias=None, eps=1e-6, kind="layer", act=None, gate=None, keep=None, ptr=None):
    n = normed(z.double(), kind, eps) * weight.double()
    n = n if bias is None else n + bias.double()
    if ptr is not None:
        plot = torch.bucketize(torch.arange(z.shape[0], device=z.device), ptr[1:].long(), right=True)
        n = n if gate is None else n * gate.double()[plot]
        n = n if keep is None else n * keep.double()[plot][:, None]
    return plain_act(r.double() + n, act).to(z.dtype)


@pytest.fixture
def plain(monkeypatch):
    """A function that puts the formulas in the kernels' place."""
    import dpcr_agb_amd.me_compat as ME
    from dpcr_agb_amd.backbones import sparse

    def replace():
        monkeypatch.setattr(ME, "row_norm_act", plain_row_norm)
        monkeypatch.setattr(ME, "row_norm_join", plain_join)
        monkeypatch.setattr(sparse, "row_norm_act", plain_row_norm)
    yield replace


def encoder(name, norm_type, **kw):
    from dpcr_agb_amd.backbones import initialize_minkowski_unet
    torch.manual_seed(3)
    model = initialize_minkowski_unet(name, 3, 2, **dict(BASE, norm_type=norm_type, **kw))
    with torch.no_grad():               # (norm weights away from one and biases away from zero)
        for k, p in model.named_parameters():
            if ".ln." in k or ".rms." in k:
                p.add_(0.1 * torch.randn_like(p))
    return model.train()


def run(model, n_points=900, plots=(0, 1, 2)):
    import dpcr_agb_amd.me_compat as ME
    from dpcr_agb_amd import synthetic
    batch = synthetic.make_sparse_batch(list(plots), n_points=n_points)
    coords = torch.cat([batch.batch[:, None].int(), batch.coords.int()], 1)
    random.seed(5)                      # (drop path)
    model.zero_grad()
    x = ME.SparseTensor(features=batch.x, coordinates=coords, device=torch.device("cuda:0"), batch_size=len(plots))
    out = model(x).F
    out.square().sum().backward()
    return out.detach().double(), {k: p.grad.detach().double() for k, p in model.named_parameters()}


# activation, options: a plain activation in the kernel, one applied behind it, block tails by modules
@pytest.mark.gpu
@pytest.mark.parametrize("name,norm_type,activation,options", [
    ("ResNet14_", "rms", "gelu", {}), ("ResNet14_", "ln", "relu", {}), ("ResNet14_", "rms", "silu", {}),
    ("ResNet50_", "rms", "relu", {}), ("SENet14", "rms", "gelu", {}), ("SENet14", "ln", "gelu", {}), ("SENet50", "rms", "gelu", {}),
    ("SENet14", "rms", "celu", {}), ("SENet14", "ln", "relu", dict(fused_tail=False))])
def test_networks_equal_the_formulas(device, plain, name, norm_type, activation, options):
    from dpcr_agb_amd.sparse_ops import KernelOptions
    model = encoder(name, norm_type, activation=activation).to(device)
    model.kernel_options = KernelOptions(fused_row_norm=True, deterministic_wgrad=True, **options)
    got, g_got = run(model)
    plain()
    want, g_want = run(model)
    assert torch.isfinite(got).all()
    assert float((got - want).abs().max() / want.abs().max()) < 1e-4
    for k in g_want:       # fp32 through up to 53 norms; a rounding of 2^-24 per value and layer leaves 1e-5 and a few times that
        if activation == "relu":
            # a value closer to zero than the two sides' difference (1e-6 of values of size one) has a gradient on one side only:
            # 2 * 0.4 * 1e-6 of the elements, whose part of a layer's gradient is the root of that in the 2-norm, 9e-4; over the
            # square root of 50 layers 6e-3, and three times that.  (Of the largest entry alone nothing can be said: behind few
            # rows one such element is all of it.  Counted once: 6 of 2.2e7 elements differ in the 50-layer network.)
            d = float((g_got[k] - g_want[k]).norm() / g_want[k].norm().clamp_min(1e-20))
            assert d < 2e-2, (k, d)
            continue
        d = float((g_got[k] - g_want[k]).abs().max() / g_want[k].abs().max().clamp_min(1e-20))
        assert d < 2e-3, (k, d)


@pytest.mark.gpu
@pytest.mark.parametrize("name,norm_type", [("SENet14", "rms"), ("ResNet14_", "ln")])
def test_networks_on_bf16_rows(device, plain, name, norm_type):
    """bf16 rows go through the kernels as they are.  Both sides round every row matrix to 2^-8; the roundings differ where a norm
    and what follows it are one pass here as there, so only in values that lie next to a rounding's edge."""
    from dpcr_agb_amd.sparse_ops import KernelOptions
    model = encoder(name, norm_type).to(device)
    model.kernel_options = KernelOptions(fused_row_norm=True, precision="bf16", bf16_activations=True)
    got, g_got = run(model)
    plain()
    want, g_want = run(model)
    a, b = (torch.cat([g[k].reshape(-1) for k in g_want]) for g in (g_got, g_want))
    assert float((got - want).abs().max() / want.abs().max()) < 5e-2
    assert float(torch.dot(a, b) / (a.norm() * b.norm())) > 0.97


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["SENet14", "ResNet50_"])
def test_layer_norm_keeps_its_kernels_unless_asked(device, monkeypatch, name):
    import dpcr_agb_amd.me_compat as ME
    from dpcr_agb_amd import norm_ops
    from dpcr_agb_amd.backbones import sparse

    def refuse(*a, **kw):
        raise AssertionError("row norm kernels without KernelOptions.fused_row_norm")
    model = encoder(name, "ln").to(device)
    for m in (ME, sparse):
        monkeypatch.setattr(m, "row_norm_act", refuse)
    monkeypatch.setattr(ME, "row_norm_join", refuse)
    calls = []
    real = norm_ops.layer_norm
    monkeypatch.setattr(norm_ops, "layer_norm", lambda x, ln: calls.append(1) or real(x, ln))
    run(model)
    assert len(calls) == sum(isinstance(m, sparse.MinkowskiLayerNorm) for m in model.modules())


@pytest.mark.gpu
def test_training_step_with_muon(device, plain):
    """A model as a user builds one: norm_type and optimiser by name.  Two steps: the gradients are those of the formulas, the
    parameters after a step those of the update's formula on the recorded gradients, and the next pass sees them."""
    from dpcr_agb_amd import synthetic
    from dpcr_agb_amd.config import MODEL_OPTIONS, Opt
    from dpcr_agb_amd.instance import MinkowskiBaselineModel
    from dpcr_agb_amd.muon_ops import matrix_shape
    torch.manual_seed(0)
    ds = synthetic.SyntheticDataset(feature_dimension=3, stat_seeds=range(10_000, 10_032))
    opt = Opt(MODEL_OPTIONS["SENet14"])
    opt["drop_path"], opt["norm_type"] = 0.0, "rms"
    model = MinkowskiBaselineModel(opt, "minkowski", ds).to(device).train()
    model.set_kernel_options(deterministic_wgrad=True)
    lr, mu, wd, clip = 2e-3, 0.9, 0.1, 0.5
    model.init_train_objects(Opt(dict(grad_clip=clip, optim=dict(optimizer=dict(
        name="Muon", params=dict(lr=lr, momentum=mu, weight_decay=wd))))))
    batch = synthetic.make_sparse_batch([0, 1, 2], n_points=1500)

    def gradients(m):
        m.zero_grad(set_to_none=True)
        m.set_input(batch, device)
        m.forward()
        m.loss.backward()
        return float(m.loss.detach()), {k: p.grad.detach().clone() for k, p in m.named_parameters()}

    momenta = {}
    for step in range(2):
        loss, grads = gradients(model)
        before = {k: p.detach().clone() for k, p in model.named_parameters()}
        model.optimizer.step()
        kinds = set()
        for k, p in model.named_parameters():
            shape = matrix_shape(p)
            kinds.add(shape is not None)
            if shape is None:
                continue
            m = momenta.setdefault(k, torch.zeros(p.shape, dtype=torch.float64, device=device))
            assert not torch.equal(p, before[k]), k
            want, momenta[k], bound = update64(before[k], grads[k], m, lr, mu, True, wd, clip)
            assert float((p.detach().double() - want).norm()) <= 2 * bound + 4 * 2.0 ** -24 * float(want.norm()), k
        assert kinds == {True, False}
    # a model that has never been stepped, with the same parameters: nothing of the earlier ones is kept anywhere
    other = MinkowskiBaselineModel(opt, "minkowski", ds).to(device).train()
    other.set_kernel_options(deterministic_wgrad=True)
    other.load_state_dict(model.state_dict())
    a, ga = gradients(model)
    b, gb = gradients(other)
    assert a == b
    plain()
    c, gc = gradients(model)
    assert abs(a - c) <= 1e-4 * abs(c)
    for k in ga:
        assert float((ga[k] - gb[k]).abs().max()) <= 1e-5 * float(gb[k].abs().max()), k
        assert float((ga[k] - gc[k]).double().abs().max() / gc[k].abs().max().clamp_min(1e-20)) < 2e-3, k


def test_options_and_names():
    from dpcr_agb_amd.backbones import initialize_minkowski_unet
    from dpcr_agb_amd.backbones.sparse import MinkowskiRMSNorm
    from dpcr_agb_amd.sparse_ops import DEFAULTS, KernelOptions
    import dpcr_agb_amd.me_compat as ME
    assert KernelOptions().fused_row_norm == DEFAULTS.fused_row_norm
    assert KernelOptions(fused_row_norm=True).replace(precision="bf16").fused_row_norm
    model = encoder("SENet14", "rms")
    keys = set(model.state_dict())
    assert {"blocks.0.0.norm.rms.weight", "blocks.1.0.norm2.rms.weight", "blocks.2.0.downsample.1.rms.weight"} <= keys
    assert not any(".rms.bias" in k for k in keys)
    assert all(ME.row_norm_form(m)["kind"] == "rms" for m in model.modules() if isinstance(m, MinkowskiRMSNorm))
    ln = encoder("ResNet14_", "ln").blocks[0][0].norm
    with KernelOptions(fused_row_norm=False):
        assert ME.row_norm_form(ln) is None
    with KernelOptions(fused_row_norm=True):
        assert ME.row_norm_form(ln)["kind"] == "layer"
    assert ME.row_norm_form(ME.MinkowskiBatchNorm(8)) is None and ME.row_norm_form(torch.nn.Identity()) is None
    with pytest.raises(NotImplementedError, match="rms"):
        initialize_minkowski_unet("ResNet14_", 3, 2, **dict(BASE, norm_type="group"))
