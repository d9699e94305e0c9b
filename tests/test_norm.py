"""Group normalisation and dropout without a GPU: the oracle's generator against published outputs, its gradients against differences,
and every refusal of the C entries and of fisr_amd/norm.py (all are decided on the host, before anything is launched)."""
import ctypes

import numpy as np
import pytest

import fisr_norm_oracle as no
from fisr_amd import lib


def test_generator_known_answers():
    """Known answers that the generator's authors publish for Philox4x32 (10 rounds; 7 rounds for the zero counter)."""
    f = lambda ctr, key, r: [int(v) for v in no.philox4x32(np.array(ctr, np.uint64), key, r)]  # noqa: E731
    assert f([0] * 4, (0, 0), 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert f([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF), 10) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert f([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0), 10) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    assert f([0] * 4, (0, 0), 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]


def test_generator_rate_and_independence():
    """The dropped share of 2^20 elements is within 5 standard deviations of t / 65536; neighbouring calls' masks agree as often as
    independent ones do (5 standard deviations again)."""
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        t = round(p * 65536) / 65536
        a, b = (no.drop_numbers(0, n, 1234567890123456789, k) < p * 65536 for k in (7, 8))
        assert abs(a.mean() - t) < 5 * np.sqrt(t * (1 - t) / n)
        both = t * t + (1 - t) * (1 - t)
        assert abs((a == b).mean() - both) < 5 * np.sqrt(both * (1 - both) / n)


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
def test_oracle_gradients_against_differences(name):
    r = np.random.default_rng(3)
    x, dy = r.standard_normal((2, 3, 2, 6)), r.standard_normal((2, 3, 2, 6))
    gamma, beta = 1 + 0.2 * r.standard_normal(6), 0.2 * r.standard_normal(6)
    fac = no.drop_factor(x.shape, 0.25, 5, 6)
    loss = lambda x, g, b: float((no.forward(x, 3, g, b, 1e-5, name, fac)[0] * dy).sum())  # noqa: E731
    for got, k in zip(no.backward(dy, x, 3, gamma, beta, 1e-5, name, fac), range(3)):
        leaf = [x, gamma, beta]
        v = r.standard_normal(leaf[k].shape)
        h = 1e-6
        hi, lo = ([q + s * h * v if j == k else q for j, q in enumerate(leaf)] for s in (1, -1))
        num = (loss(*hi) - loss(*lo)) / (2 * h)
        # third derivatives are O(10) here: h^2 * 10 = 1e-11; rounding 1e-16 * 30 / h = 3e-9
        assert abs(num - float((got * v).sum())) < 1e-7, name


P, Q = 4096, 8192          # stand-ins for device pointers: every call below is refused before they are used


def _gn(**kw):
    a = dict(x=P, x_cs=8, gamma=None, beta=None, y=P, y_cs=8, st=P, n=1, h=2, w=2, c=8, g=2, eps=1e-5, act=0, drop=None, type=0, ws=P, nb=1 << 20)
    a.update(kw)
    return lib.lib().fisr_train_groupnorm(*a.values(), None)


def _gb(**kw):
    a = dict(x=P, x_cs=8, dy=P, dy_cs=8, gamma=None, beta=None, st=P, dx=P, dx_cs=8, dg=None, db=None, acc=0, n=1, h=2, w=2, c=8, g=2, act=0, drop=None,
             type=0, ws=P, nb=1 << 20)
    a.update(kw)
    return lib.lib().fisr_train_groupnorm_bwd(*a.values(), None)


def _drop(p, counter=None):
    return ctypes.byref(lib.DropoutDesc(p, 1, 2, counter))


BAD = [dict(x=None), dict(st=None), dict(n=0), dict(h=0), dict(w=-1), dict(c=0), dict(g=0), dict(g=3), dict(x_cs=7), dict(x_cs=-8), dict(act=4), dict(act=-1),
       dict(type=3), dict(type=-1), dict(ws=P + 4), dict(x=P + 2), dict(x=P + 1, type=1), dict(gamma=P + 2), dict(st=P + 1),
       dict(h=1 << 15, w=(1 << 15) + 1), dict(n=(1 << 20) + 1), dict(n=1 << 20, g=8), dict(c=(1 << 16) + 2, x_cs=1 << 17),
       dict(drop=_drop(-0.1)), dict(drop=_drop(1.1)), dict(drop=_drop(float("nan"))), dict(drop=_drop(0.5, P + 4))]


@pytest.mark.parametrize("kw", BAD + [dict(y=None), dict(y_cs=7), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))], ids=str)
def test_groupnorm_refuses(kw):
    lib.build()
    assert _gn(**kw) == -1
    assert b"groupnorm" in lib.lib().fisr_last_error(None)


@pytest.mark.parametrize("kw", BAD + [dict(dy=None), dict(dx=None), dict(dy_cs=4), dict(dx_cs=0), dict(dy=P + 2), dict(dg=P + 1), dict(db=P + 2)], ids=str)
def test_groupnorm_backward_refuses(kw):
    lib.build()
    assert _gb(**kw) == -1
    assert b"groupnorm_bwd" in lib.lib().fisr_last_error(None)


def test_workspace_of_the_wrong_size_is_refused():
    L = lib.lib()
    need = [L.fisr_train_groupnorm_workspace_bytes(2, 200, 300, 24, 4, b) for b in (0, 1)]
    assert 0 < need[0] < need[1]
    assert L.fisr_train_groupnorm_workspace_bytes(0, 2, 2, 8, 2, 0) == 0 and L.fisr_train_groupnorm_workspace_bytes(1, 2, 2, 8, 3, 0) == 0
    assert _gn(n=2, h=200, w=300, c=24, g=4, x_cs=24, y_cs=24, nb=need[0] - 1) == -5
    assert _gn(n=2, h=200, w=300, c=24, g=4, x_cs=24, y_cs=24, ws=None) == -5
    assert _gb(ws=None) == -5
    assert _gb(n=2, h=200, w=300, c=24, g=4, x_cs=24, dy_cs=24, dx_cs=24, nb=need[1] - 1) == -5


def test_dropout_refuses():
    f = lib.lib().fisr_train_dropout
    ok = _drop(0.5)
    assert f(P, None, P, 0, ok, 0, None) == 0                      # nothing to do
    for a in ((None, None, P, 8, ok, 0), (P, None, None, 8, ok, 0), (P, None, P, 8, ok, 5), (P + 2, None, P, 8, ok, 0), (P, P + 1, P, 8, ok, 1),
              (P, None, P, 8, _drop(-1e-9), 0), (P, None, P, 8, _drop(float("nan")), 0), (P, None, P, 8, _drop(0.5, P + 1), 0)):
        assert f(*a, None) == -1


def test_pointers_that_are_no_device_memory_are_refused():
    """Whole calls with pointers to nothing, and to host memory: refused before a launch."""
    host = ctypes.create_string_buffer(1 << 16)
    for p in (P, ctypes.addressof(host) // 64 * 64 + 64):
        assert _gn(x=p, y=p, st=p, ws=p) == -1 and b"memory" in lib.lib().fisr_last_error(None)
        assert _gb(x=p, dy=p, dx=p, st=p, ws=p) == -1 and b"memory" in lib.lib().fisr_last_error(None)
        assert lib.lib().fisr_train_dropout(p, None, p, 8, _drop(0.5), 0, None) == -1


def test_outputs_across_an_input_are_refused():
    import torch
    from fisr_amd import norm
    b = torch.zeros(2, 3, 4, 24)
    cs = lambda t: norm._pixel_stride(t, "t")  # noqa: E731
    far = torch.zeros(2, 3, 4, 8)
    x = b[..., 4:12]
    for ok in (x, b[..., 12:20], b[..., :4][..., :4], far):
        if ok.shape == x.shape:
            norm._apart(ok, cs(ok), x, cs(x), "out")
    for bad in (b[..., 8:16], b[..., 0:8], b[..., 3:11], b.view(-1)[8:8 + far.numel()].view(far.shape)):
        with pytest.raises(ValueError, match="overlaps"):
            norm._apart(bad, cs(bad), x, cs(x), "out")
    flat = torch.zeros(100)
    with pytest.raises(ValueError, match="overlaps"):
        norm._apart(flat[1:51], 50, flat[:50], 50, "out")
    norm._apart(flat[50:], 50, flat[:50], 50, "out")


def test_python_entries_refuse():
    import torch
    from fisr_amd import norm
    x = torch.zeros(1, 2, 2, 8)
    with pytest.raises(lib.FisrError, match="no CPU fallback"):
        norm.group_norm(x, 2)
    with pytest.raises(lib.FisrError, match="no CPU fallback"):
        norm.dropout(x, norm.Dropout(0.5, 1))
    with pytest.raises(ValueError, match="N, H, W, C"):
        norm.group_norm(x[0], 2)
    with pytest.raises(ValueError, match="bfloat16"):
        norm.group_norm(x.double(), 2)
    for p in (-0.5, 1.5, float("nan")):
        with pytest.raises(ValueError, match="not in"):
            norm.Dropout(p, 1)
    with pytest.raises(ValueError, match="int64"):
        norm.Dropout(0.5, 1, counter=torch.zeros(1))
    # pixel strides: dense, a channel range, one pixel only; refused: transposed channels, cropped rows
    wide = torch.zeros(2, 3, 4, 24)
    assert norm._pixel_stride(wide, "x") == 24 and norm._pixel_stride(wide[..., 8:16], "x") == 24
    assert norm._pixel_stride(wide[:1, :1, :1, 4:8], "x") == 4 or norm._pixel_stride(wide[:1, :1, :1, 4:8], "x") >= 4
    assert norm._pixel_stride(wide[:, :1, :1, :8], "x") == 288
    for bad in (wide.permute(0, 3, 1, 2), wide[:, :, :2], wide[:, :2], wide[..., ::2], wide[:, ::2], wide[:1, :1, :1].expand(2, 3, 4, 24)):
        with pytest.raises(ValueError, match="one stride"):
            norm._pixel_stride(bad, "x")


@pytest.mark.parametrize("call,name,said", [(_gn, "gamma", "gamma"), (_gn, "beta", "beta"), (_gb, "gamma", "gamma"), (_gb, "beta", "beta"), (_gb, "dg", "dgamma"),
                                            (_gb, "db", "dbeta"), (_gn, "st", "mean_rstd"), (_gb, "st", "mean_rstd")])
def test_every_operand_that_is_no_device_memory_is_refused(call, name, said):
    """A call's pointers are asked for one by one, the parameters and their gradients first: the first that is no memory of a GPU is named, before
    anything is launched."""
    host = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(host) // 64 * 64 + 64
    assert call(**{name: p}) == -1 and lib.lib().fisr_last_error(None).decode().endswith(f": {said} is not memory of a GPU")


def test_a_counter_in_host_memory_is_refused():
    host = (ctypes.c_uint64 * 2)()
    p = ctypes.addressof(host)
    assert lib.lib().fisr_train_dropout(P, None, P, 8, _drop(0.5, p), 0, None) == -1 and b"d_counter is not memory" in lib.lib().fisr_last_error(None)
    for call in (_gn, _gb):
        assert call(drop=_drop(0.5, p)) == -1 and b"d_counter is not memory" in lib.lib().fisr_last_error(None)


def test_strides_and_places_exactly():
    """The stride of a single pixel's channels is their number, whatever buffer they are a range of; ranges of channels before x, behind it and
    across it."""
    import torch
    from fisr_amd import norm
    wide = torch.zeros(2, 3, 4, 24)
    assert norm._pixel_stride(wide[:1, :1, :1, 4:8], "x") == 4
    x = wide[..., 12:20]
    for ok in (wide[..., 0:8], wide[..., 4:12], x):
        assert ok.shape == x.shape
        norm._apart(ok, 24, x, 24, "out")
    for bad in (wide[..., 5:13], wide[..., 13:21], wide[..., 16:24]):
        with pytest.raises(ValueError, match="overlaps"):
            norm._apart(bad, 24, x, 24, "out")


def test_the_build_entry_compiles_what_is_built_already(monkeypatch):
    """build() is what says that the sources compile, so it compiles them where a library is there too."""
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(lib, "build", lambda force=False, verbose=False: (calls.append(force), lib.SO_PATH)[1])
    entry.build()
    assert calls == [True]
