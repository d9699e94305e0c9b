"""Group normalisation and dropout on the training tape (fisr_amd/train.py), as they are used together: a normalised residual block between
two of the network's convs, dropout in the network's own blocks, and `--phase train --dropout`."""
import numpy as np
import pytest

import fisr_norm_oracle as no

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from fisr_amd import norm, train, weights
    return torch, norm, train, weights


def _rel(a, b):
    a, b = (np.asarray(v.detach().cpu() if hasattr(v, "cpu") else v, np.float64) for v in (a, b))
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("hw", [(7, 9), (24, 24)])
def test_normalised_residual_block_vs_autograd(env, hw):
    """y = x + drop(conv1(drop(silu(gn2(conv0(silu(gn1(x)))))))): output and every gradient against torch autograd in float64 on the CPU.
    float32 sums of up to 576 products a pixel and 4608 pixels a weight, no kinks: relative errors of 2e-5 as the other adjoints' tests."""
    torch, norm, train, weights = env
    import torch.nn.functional as F
    h, w = hw
    net = train.TrainNet(weights.synthetic_weights(3))
    names = ["FISRnet/level_1/enc/level_0/res_block/0/conv/%d" % k for k in (0, 1)]
    r = np.random.default_rng(h)
    x = torch.from_numpy(r.standard_normal((2, h, w, 64)).astype(np.float32)).cuda()
    gy = torch.from_numpy(r.standard_normal((2, h, w, 64)).astype(np.float32)).cuda()
    par = [torch.from_numpy((m + 0.2 * r.standard_normal(64)).astype(np.float32)).cuda() for m in (1, 0, 1, 0)]
    gpar = [torch.zeros(64, device="cuda") for _ in range(4)]
    d1, d2 = norm.Dropout(0.2, 11, 1), norm.Dropout(0.1, 11, 2)
    net.zero_grad()
    a = net.group_norm(x, 8, par[0], par[1], gpar[0], gpar[1], act="silu")
    b = net.conv(names[0], a)
    c = net.group_norm(b, 4, par[2], par[3], gpar[2], gpar[3], act="silu", drop=d1)
    e = net.conv(names[1], c)
    y = net.dropout(e, d2, residual=x)
    seen = {}
    acc = net._acc
    net._acc = lambda grads, t, g: (acc(grads, t, g), seen.update({t.data_ptr(): grads[t.data_ptr()]}))[0]
    net.backward([(y, gy.clone())])
    torch.cuda.synchronize()
    # ---- float64
    leaf = lambda t: t.detach().cpu().double().requires_grad_(True)  # noqa: E731
    xr, pr = leaf(x), [leaf(t) for t in par]
    wr = [leaf(net.convs[n].w) for n in names]
    br = [leaf(net.convs[n].b) for n in names]
    conv = lambda v, k: F.conv2d(v.permute(0, 3, 1, 2), wr[k].permute(3, 2, 0, 1), br[k], padding=1).permute(0, 2, 3, 1)  # noqa: E731

    def gn(v, g, gamma, beta):
        u = v.reshape(2, h * w, g, 64 // g)
        m = u.mean(dim=(1, 3), keepdim=True)
        s = ((u - m) ** 2).mean(dim=(1, 3), keepdim=True)
        return ((u - m) / torch.sqrt(s + 1e-5)).reshape(2, h, w, 64) * gamma + beta

    f1, f2 = (torch.from_numpy(no.drop_factor((2, h, w, 64), p, 11, k)) for p, k in ((0.2, 1), (0.1, 2)))
    yr = xr + conv(F.silu(gn(conv(F.silu(gn(xr, 8, pr[0], pr[1])), 0), 4, pr[2], pr[3])) * f1, 1) * f2
    yr.backward(gy.cpu().double())
    assert _rel(y, yr.detach()) < 2e-5
    assert _rel(seen[x.data_ptr()], xr.grad) < 2e-5
    for got, ref in zip(gpar, pr):
        assert _rel(got, ref.grad) < 2e-5
    for n, wt, bt in zip(names, wr, br):
        assert _rel(net.convs[n].gw, wt.grad) < 2e-5 and _rel(net.convs[n].gb, bt.grad) < 2e-5


def _batch(train):
    import fisr_train_oracle as fo
    return train.to_device_batch(fo.synthetic_batch(11, 1, 32, 32))


def test_dropout_of_zero_is_the_network_as_it_was(env):
    torch, norm, train, weights = env
    W = weights.synthetic_weights(2020)
    preds = []
    for net in (train.TrainNet(W), train.TrainNet(W, dropout=0.0, dropout_seed=5)):
        net.keep_preds = True                                     # (the predictions: the loss' sums are atomic, in no fixed order)
        net.loss_and_grads(_batch(train))
        preds.append([p for window in net.last_preds for p in window])
    assert len(preds[0]) == 12 and all(torch.equal(a, b) for a, b in zip(*preds))
    for p in (-0.1, 1.0, 2.0):
        with pytest.raises(ValueError, match="dropout"):
            train.TrainNet(W, dropout=p)


def test_dropout_in_the_network(env):
    """Masks are a function of (seed, step, block): the same step gives the same loss, another step or seed another one, `training` off the
    loss without dropout; and the gradient agrees with a difference of the loss along itself.  Loss terms are float32 sums of 9216 and more
    squares (1e-6 relative); the step along the gradient changes the loss by 1 %, so the difference is good to 1e-4 of itself and the
    curvature along it, which central differences cancel to second order, and the relus' kinks make up the rest of the 3 %."""
    torch, norm, train, weights = env
    W = weights.synthetic_weights(2020)
    batch = _batch(train)
    net = train.TrainNet(W, dropout=0.2, dropout_seed=7)
    net.zero_grad()
    l0, _ = net.loss_and_grads(batch)
    g = net.gflat.clone()
    net.zero_grad()
    l1, _ = net.loss_and_grads(batch)
    assert abs(l0 - l1) <= 1e-6 * abs(l0)                         # (the loss kernel's sums are atomic)
    w0 = net.wflat.clone()
    t = 0.005 * l0 / float((g.double() ** 2).sum())
    side = []
    for s in (1, -1):
        net.wflat.copy_(w0 + s * t * g)
        net.repack()
        side.append(net.loss_and_grads(batch)[0])
    assert abs((side[0] - side[1]) / (2 * t) / float((g.double() ** 2).sum()) - 1) < 0.03
    net.wflat.copy_(w0)
    net.repack()
    net.step_count += 1
    l2, _ = net.loss_and_grads(batch)
    net.training = False
    l3, _ = net.loss_and_grads(batch)
    plain, _ = train.TrainNet(W).loss_and_grads(batch)
    other, _ = train.TrainNet(W, dropout=0.2, dropout_seed=8).loss_and_grads(batch)
    assert abs(l2 - l0) > 1e-5 * l0 and abs(other - l0) > 1e-5 * l0 and abs(plain - l0) > 1e-5 * l0
    assert abs(l3 - plain) <= 1e-6 * plain


def test_phase_train_with_dropout(env, tmp_path):
    """The command trains with dropout and writes the same variables as without; they differ from a run without it."""
    torch, norm, train, weights = env
    from fisr_amd import main
    W = []
    for k, extra in enumerate((["--dropout", "0.2"], [])):
        d = str(tmp_path / str(k))
        assert main.main(["--phase", "train", "--synthetic_train", "4", "--epoch", "1", "--batch_size", "2", "--val_data_size", "2", "--val_batch_size", "2",
                          "--lr_type", "no_decay", "--checkpoint_dir", d + "/ck", "--text_dir", d + "/tx", "--log_dir", d + "/lg", "--test_img_dir", d + "/ti"] + extra) == 0
        path, kind, step = weights.find_checkpoint(d + "/ck", "FISRnet_exp1")
        assert step == 1
        W.append(weights.load_weights(path, kind))
    assert sorted(W[0]) == sorted(W[1]) and any(not np.array_equal(W[0][k], W[1][k]) for k in W[0])


def test_batches_of_one_step_draw_masks_of_their_own(env):
    """Gradients accumulated over two batches before a step: the second batch's masks are not the first one's (the same batch twice gives
    another loss and other gradients), and after zero_grad() or with weights packed again the numbers start where they did.  The loss' and the
    gradients' sums are atomic: 1e-6 of the loss, and 1e-3 of the gradients' norm, which masks of their own change by far more."""
    torch, norm, train, weights = env
    batch = _batch(train)
    net = train.TrainNet(weights.synthetic_weights(2020), dropout=0.2, dropout_seed=7)
    net.zero_grad()
    l0, _ = net.loss_and_grads(batch)
    g0 = net.gflat.clone()
    l1, _ = net.loss_and_grads(batch)
    g1 = net.gflat - g0
    assert abs(l1 - l0) > 1e-5 * l0 and float((g1 - g0).norm()) > 0.02 * float(g0.norm())
    net.zero_grad()
    l2, _ = net.loss_and_grads(batch)
    assert abs(l2 - l0) <= 1e-6 * l0 and float((net.gflat - g0).norm()) < 1e-3 * float(g0.norm())
    net.repack()
    l3, _ = net.loss_and_grads(batch)
    assert abs(l3 - l0) <= 1e-6 * l0


def test_normalisation_on_the_tape_without_parameters(env):
    """No gamma and beta, or gradients of one that are not wanted: dx is that of ones and zeros, and the wanted gradient is what it was."""
    torch, norm, train, weights = env
    net = train.TrainNet(weights.synthetic_weights(3))
    r = np.random.default_rng(5)
    x, gy = (torch.from_numpy(r.standard_normal((2, 7, 9, 64)).astype(np.float32)).cuda() for _ in range(2))
    one, zero = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    got = []
    acc = net._acc
    net._acc = lambda grads, t, g: (got.append(g.clone()), acc(grads, t, g))
    for gamma, beta, wants in ((one, zero, (1, 1)), (None, None, (0, 0)), (one, zero, (1, 0)), (one, zero, (0, 1))):
        grads = [torch.zeros(64, device="cuda") if k else None for k in wants]
        y = net.group_norm(x, 8, gamma, beta, *grads, act="silu")
        net.backward([(y, gy)])
        if wants == (1, 1):
            want = grads
        assert torch.equal(got[-1], got[0]) and all(g is None or torch.equal(g, w) for g, w in zip(grads, want))
    assert len(got) == 4


def test_the_command_drops_in_training_and_not_in_validation(env, tmp_path, monkeypatch):
    """--dropout P is the P of the network that the command trains: each of its training passes has a dropout in every residual block, its
    validation passes have none, and without the option there is none at all."""
    torch, norm, train, weights = env
    from fisr_amd import main
    nets = []

    class Seen(train.TrainNet):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            self.passes = []                                    # (training, dropouts)
            nets.append(self)

        def model(self, x):
            self.passes.append([self.training, 0])
            return super().model(x)

        def dropout(self, x, drop, residual=None):
            assert drop.p == 0.2 and residual is None
            self.passes[-1][1] += 1
            return super().dropout(x, drop, residual)

    monkeypatch.setattr(train, "TrainNet", Seen)
    blocks = sum(name.endswith("/conv/1") and "res_block" in name for name, _, _ in weights.conv_specs())
    assert blocks > 10
    for k, extra in enumerate((["--dropout", "0.2"], [])):
        d = str(tmp_path / str(k))
        assert main.main(["--phase", "train", "--synthetic_train", "4", "--epoch", "1", "--batch_size", "2", "--val_data_size", "2", "--val_batch_size", "2",
                          "--lr_type", "no_decay", "--checkpoint_dir", d + "/ck", "--text_dir", d + "/tx", "--log_dir", d + "/lg", "--test_img_dir", d + "/ti"] + extra) == 0
    assert [n.dropout_p for n in nets] == [0.2, 0.0]
    for net, drops in zip(nets, (blocks, 0)):
        assert {t for t, _ in net.passes} == {True, False}
        assert all(n == (drops if training else 0) for training, n in net.passes), net.passes
