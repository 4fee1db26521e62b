"""Layer operators without a GPU: the generator's published answers, and every refusal of the C entry points (all of
them come before the device is touched, so the addresses here are never read)."""
import ctypes as C
import inspect

import numpy as np
import pytest

torch = pytest.importorskip("torch")   # before libepi.so: the two share torch's HIP runtime

from epidemicsimulator_amd import _capi  # noqa: E402
from oracle import layers_ref as R  # noqa: E402

BAD, DEVICE, UNSUPPORTED = _capi.EPI_ERR_BAD_ARGUMENT, _capi.EPI_ERR_DEVICE, _capi.EPI_ERR_UNSUPPORTED


@pytest.mark.parametrize("counter, key, want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_known_answers(counter, key, want):
    assert R.philox4x32(counter, key) == list(want)


def test_draws_are_the_halves_of_the_words():
    d = R.draws(3, 19, 0x299F31D0A4093822, 0x0370734413198A2E, first_row=0x85A308D1)
    for r in range(3):
        for c in range(19):
            w = R.philox4x32((c // 8, 0x85A308D1 + r, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0))
            assert int(d[r, c]) == (w[c % 8 // 2] >> (16 * (c % 2))) & 0xFFFF


def test_mask_has_its_probability_and_no_lines():
    """p = 0.3 over 2^20 units: the share dropped within 6 deviations of its mean, and so that of each row and column."""
    n = 1024
    dropped = R.factors(n, n, 0.3, 11, 5) == 0
    p = R.threshold(0.3) / 65536
    for share, count in ((dropped.mean(), n * n), (dropped.mean(0), n), (dropped.mean(1), n)):
        assert np.all(np.abs(share - p) < 6 * np.sqrt(p * (1 - p) / count))


def desc(**kw):
    d = _capi.LayerDesc(rows=4, cols=8, x_stride=8, y_stride=8, dy_stride=8, eps=1e-5, dropout=0.0, seed=0, offset=0,
                        offset_dev=None, dtype=1, device=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


ADDR = [0x10000 * (k + 1) for k in range(12)]   # apart and aligned; never read
N = None


def call(fn, *args):
    L = _capi.lib()
    return getattr(L, fn)(*args)


def refused(status, fn, *args):
    assert call(fn, *args) == status
    assert _capi.last_error()


WRONG_DESCS = [dict(dtype=4), dict(dtype=-1), dict(rows=-1), dict(cols=0), dict(cols=-3), dict(dropout=-0.1),
               dict(dropout=1.0001), dict(dropout=float("nan")), dict(offset_dev=0x1004)]


@pytest.mark.parametrize("wrong", WRONG_DESCS)
def test_wrong_descriptors_are_refused(wrong):
    d = C.byref(desc(**wrong))
    refused(BAD, "epi_dropout", d, ADDR[0], ADDR[1], N)
    refused(BAD, "epi_layer_norm_forward", d, ADDR[0], ADDR[1], ADDR[2], ADDR[3], ADDR[4], ADDR[5], N)
    refused(BAD, "epi_layer_norm_backward", d, *ADDR[:9], 0, N)
    refused(BAD, "epi_layer_norm_backward_workspace", d, C.byref(C.c_size_t()))


@pytest.mark.parametrize("size", [dict(rows=1 << 31), dict(cols=1 << 31, x_stride=1 << 31, y_stride=1 << 31)])
def test_sizes_beyond_the_counter_are_refused(size):
    refused(UNSUPPORTED, "epi_dropout", C.byref(desc(**size)), ADDR[0], ADDR[1], N)


def test_null_arguments_are_refused():
    d = C.byref(desc())
    refused(BAD, "epi_dropout", None, ADDR[0], ADDR[1], N)
    refused(BAD, "epi_dropout", d, N, ADDR[1], N)
    refused(BAD, "epi_dropout", d, ADDR[0], N, N)
    refused(BAD, "epi_layer_norm_forward", d, N, N, N, ADDR[3], N, N, N)
    refused(BAD, "epi_layer_norm_forward", d, ADDR[0], N, N, N, N, N, N)
    refused(BAD, "epi_layer_norm_forward", d, ADDR[0], N, N, ADDR[3], ADDR[4], N, N)      # mean without rstd
    refused(BAD, "epi_layer_norm_forward", d, ADDR[0], N, N, ADDR[3], N, ADDR[4], N)
    for k in (0, 1, 3, 4):                                                                # x, dy, mean, rstd
        args = list(ADDR[:9]); args[k] = N
        refused(BAD, "epi_layer_norm_backward", d, *args, 0, N)
    refused(BAD, "epi_layer_norm_backward_workspace", d, None)


@pytest.mark.parametrize("wrong", [dict(x_stride=-1), dict(y_stride=7), dict(y_stride=0), dict(x_stride=1 << 40)])
def test_wrong_strides_are_refused(wrong):
    refused(BAD, "epi_dropout", C.byref(desc(**wrong)), ADDR[0], ADDR[1], N)
    refused(BAD, "epi_layer_norm_forward", C.byref(desc(**wrong)), ADDR[0], N, N, ADDR[1], N, N, N)


@pytest.mark.parametrize("name", ["x_stride", "y_stride"])
def test_rows_beyond_the_address_space_are_refused(name):
    """2^31 - 1 rows, 2^38 elements apart, end behind 2^63 bytes: their extent is not taken modulo 2^64.  2^31 - 1 rows
    2^29 apart end below 2^63: the call goes on to the overlap of x and y."""
    rows = (1 << 31) - 1
    x, y = (1 << 20, 1 << 40) if name == "x_stride" else (1 << 40, 1 << 20)
    for stride, why in ((1 << 38, "row stride"), ((1 << 40) - 1, "row stride"), (1 << 62, "row stride"), (1 << 29, "overlap")):
        d = desc(rows=rows, **{name: stride})
        refused(BAD, "epi_dropout", C.byref(d), x, y, N)
        assert why in _capi.last_error()
        refused(BAD, "epi_layer_norm_forward", C.byref(d), x, N, N, y, N, N, N)
        assert why in _capi.last_error()


def test_misaligned_arrays_are_refused():
    d = C.byref(desc())
    refused(BAD, "epi_dropout", d, ADDR[0] + 2, ADDR[1], N)
    refused(BAD, "epi_dropout", d, ADDR[0], ADDR[1] + 1, N)
    for k in range(6):
        args = list(ADDR[:6]); args[k] += 2
        refused(BAD, "epi_layer_norm_forward", d, *args, N)
    for k in range(9):
        args = list(ADDR[:9]); args[k] += 2
        refused(BAD, "epi_layer_norm_backward", d, *args, 1 << 20, N)


def test_overlapping_arrays_are_refused():
    d = C.byref(desc())
    refused(BAD, "epi_dropout", d, ADDR[0], ADDR[0] + 32, N)
    refused(BAD, "epi_dropout", C.byref(desc(y_stride=9)), ADDR[0], ADDR[0], N)           # in place with other strides
    for k in (1, 2, 4, 5):                                                                # y on weight, bias, mean, rstd
        args = list(ADDR[:6]); args[k] = ADDR[3] + 4
        refused(BAD, "epi_layer_norm_forward", d, *args, N)
    args = list(ADDR[:6]); args[5] = args[4] + 4                                          # mean on rstd
    refused(BAD, "epi_layer_norm_forward", d, *args, N)
    for o in (5, 6, 7):                                                                   # dx, dweight, dbias on inputs
        for i in range(5):
            args = list(ADDR[:9]); args[o] = args[i]
            refused(BAD, "epi_layer_norm_backward", d, *args, 1 << 20, N)
    args = list(ADDR[:9]); args[7] = args[6] + 4
    refused(BAD, "epi_layer_norm_backward", d, *args, 1 << 20, N)


def test_negative_eps_is_refused():
    for eps in (-1e-9, float("nan")):
        refused(BAD, "epi_layer_norm_forward", C.byref(desc(eps=eps)), ADDR[0], N, N, ADDR[1], N, N, N)


def workspace(**kw):
    n = C.c_size_t(1)
    assert call("epi_layer_norm_backward_workspace", C.byref(desc(**kw)), C.byref(n)) == 0
    return n.value


def test_a_workspace_that_is_too_small_is_refused():
    big = dict(rows=100000, cols=129, x_stride=129, y_stride=129, dy_stride=129)
    need = workspace(**big)
    assert need > 0
    far = [0x1_0000_0000 * (k + 1) for k in range(9)]
    refused(BAD, "epi_layer_norm_backward", C.byref(desc(**big)), *far, need - 1, N)
    refused(BAD, "epi_layer_norm_backward", C.byref(desc(**big)), *far[:8], N, need, N)


def test_valid_arguments_reach_the_device_check():
    if _capi.lib().epi_device_count() > 0:
        pytest.skip("has a GPU")
    d = C.byref(desc())
    refused(DEVICE, "epi_dropout", d, ADDR[0], ADDR[1], N)
    refused(DEVICE, "epi_dropout", d, ADDR[0], ADDR[0], N)                                # in place
    refused(DEVICE, "epi_layer_norm_forward", d, ADDR[0], N, N, ADDR[1], N, N, N)
    refused(DEVICE, "epi_layer_norm_backward", d, *ADDR[:9], 1 << 20, N)
    refused(DEVICE, "epi_layer_norm_backward", C.byref(desc(x_stride=0, dy_stride=0)), *ADDR[:9], 1 << 20, N)


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    from epidemicsimulator_amd import layers
    x = torch.zeros(3, 8)
    for f in (lambda: layers.dropout(x, 0.1, 1), lambda: layers.layer_norm(x), lambda: layers.layer_norm_forward(x),
              lambda: layers.layer_norm_backward(x, x, None, x[:, 0], x[:, 0]), lambda: layers.layer_norm([1.0, 2.0])):
        with pytest.raises(_capi.EpiError) as e:
            f()
        assert e.value.status == BAD


def test_tangents_are_refused():
    """The tangent of a dual tensor would be lost and read as zero; seen before anything else, so without a GPU too."""
    import torch.autograd.forward_ad as forward_ad
    from epidemicsimulator_amd import layers
    x, w = torch.ones(3, 8), torch.ones(8)
    with forward_ad.dual_level():
        t, v = forward_ad.make_dual(x, torch.ones(3, 8)), forward_ad.make_dual(w, torch.ones(8))
        for f in (lambda: layers.dropout(t, 0.1, 1), lambda: layers.layer_norm(t), lambda: layers.layer_norm(x, v), lambda: layers.layer_norm(x, None, v)):
            with pytest.raises(_capi.EpiError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(_capi.EpiError, match="forward-mode"):
                f()
            with forward_ad._set_fwd_grad_enabled(False), pytest.raises(_capi.EpiError, match="on the GPU only"):
                f()


def test_tensors_without_memory_are_refused():
    """Fake tensors of a GPU, whose views have addresses next to zero: refused before anything is enqueued."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from epidemicsimulator_amd import layers
    with FakeTensorMode():
        x, w, m = (torch.empty(n, device="cuda:0") for n in ((6, 8), 9, 5))
        off = torch.empty(2, device="cuda:0", dtype=torch.int64)
        for f in (lambda: layers.dropout(x, 0.1, 1), lambda: layers.dropout(x[1:], 0.1, 1), lambda: layers.layer_norm(x[1:]), lambda: layers.layer_norm(x[1:], w[1:]),
                  lambda: layers.layer_norm_forward(x[1:], None, w[1:]), lambda: layers.dropout(x[1:], 0.1, 1, off[1]),
                  lambda: layers.layer_norm_backward(x[1:], x[:5], None, m, m)):
            with pytest.raises(_capi.EpiError, match="no memory"):
                f()


def test_two_hip_runtimes_are_refused():
    """libepi.so loaded before torch: the binding says so instead of mixing the two (in a process of its own)."""
    import subprocess
    import sys
    code = ("import epidemicsimulator_amd as E; E.lib()\n"
            "try:\n    from epidemicsimulator_amd import layers\n"
            "except ImportError as e:\n    assert 'two HIP runtimes' in str(e)\n"
            "else:\n    assert len(layers._hip_runtimes()) == 1\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_public_names_are_documented():
    from epidemicsimulator_amd import layers
    for name in layers.__all__:
        assert inspect.getdoc(getattr(layers, name))


def layouts():
    """Tensors of two to four dimensions over small storages: permuted, sliced, expanded, single columns and rows, none."""
    import itertools
    for sizes in ((5, 8), (6, 1), (1, 8), (4, 3, 8), (2, 3, 1), (1, 5, 7), (3, 1, 9), (0, 3, 8), (3, 0, 8), (2, 3, 4, 5), (2, 1, 3, 8), (1, 3, 1, 2), (2, 2, 2, 1)):
        t = torch.arange(float(np.prod(sizes))).view(sizes)
        views = [t.permute(order) for order in itertools.permutations(range(t.dim()))]
        views += [t[tuple(slice(None, None, step) for step in steps)] for steps in itertools.product((1, 2), repeat=t.dim())]
        views += [t.narrow(d, 1, t.shape[d] - 1) for d in range(t.dim()) if t.shape[d] > 1]
        for v in views:
            yield v
            for ones in itertools.product((False, True), repeat=v.dim()):   # one index of some dimensions, expanded again
                if v.numel():
                    w = v[tuple(slice(0, 1) if one else slice(None) for one in ones)]
                    yield w
                    yield w.expand([4 if n == 1 else n for n in w.shape])
                    yield w.expand([3 if one else n for one, n in zip(ones, w.shape)])
            for d in range(v.dim() + 1):
                u = v.unsqueeze(d)
                yield u.expand([3 if k == d else n for k, n in enumerate(u.shape)])


def test_rows_are_read_where_they_lie():
    """The distance the binding answers, taken over the tensor's storage, gives the tensor's rows (as_strided refuses what
    lies outside the storage); no answer means a copy, which contiguous tensors never need."""
    from epidemicsimulator_amd import layers
    answers = set()
    for t in layouts():
        step = layers._layers.row_distance(t)
        answers.add((t.dim(), step is None, step == 0))
        if step is None:
            assert not t.is_contiguous()
            continue
        rows = t.numel() // t.shape[-1] if t.shape[-1] else 0
        got = t.as_strided((rows, t.shape[-1]), (step, 1))
        assert torch.equal(got, t.contiguous().view(rows, t.shape[-1])), (t.shape, t.stride(), step)
    for dims in (2, 3, 4):
        assert (dims, True, False) in answers and (dims, False, True) in answers and (dims, False, False) in answers


@pytest.mark.parametrize("sizes, strides, want", [
    ((4, 3, 128), (128, 0, 1), None), ((4, 3, 2, 128), (128, 0, 0, 1), None), ((4, 3, 128), (0, 128, 1), None), ((4, 3, 128), (0, 0, 1), 0),
    ((4, 3, 128), (0, 0, 0), None), ((4, 3, 1), (1, 0, 0), None), ((4, 3, 128), (600, 200, 1), 200), ((4, 1, 128), (128, 0, 1), 128), ((4, 0, 8), (3, 7, 1), 8)])
def test_expanded_dimensions_in_the_middle_are_copied(sizes, strides, want):
    from epidemicsimulator_amd import layers
    assert layers._layers.row_distance(torch.zeros(4000).as_strided(sizes, strides)) == want


def test_rows_of_a_number_are_refused():
    from epidemicsimulator_amd import layers
    with pytest.raises(ValueError):
        layers._layers.row_distance(torch.tensor(1.0))


@pytest.mark.parametrize("installed", [True, False])
def test_build_asks_for_the_binding_where_torch_is_installed(monkeypatch, installed):
    """The library builds without torch, and then nothing loads the binding that was not built."""
    import importlib.util
    import __graft_entry__ as entry
    commands, found = [], importlib.util.find_spec
    monkeypatch.setattr(entry.subprocess, "check_call", lambda command, **kw: commands.append(" ".join(command)))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: found(name, *a) if installed or name != "torch" else None)
    entry.build()
    assert any("csrc" in c for c in commands)
    assert any("layers" in c for c in commands) == installed
