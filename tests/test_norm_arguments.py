"""What layer norm and dropout refuse, and the generator behind the masks: no GPU needed."""
import ctypes

import numpy as np
import pytest
import torch

import compressgnn_runtime as rt
from compressgnn_amd import abi
from CompressgnnDropout import Compressgnn_Dropout, dropout
from CompressgnnNorm import Compressgnn_LayerNorm, layer_norm, norm_act_dropout
from rows_reference import factors, kept_share, mask, philox

EINVAL, EWORKSPACE, EUNSUPPORTED = 1, 2, 4


def test_generator_gives_the_published_numbers():
    """The known answers of Philox4x32-10 published with it (Random123): zeros, ones, digits of pi."""
    ones = 0xFFFFFFFF
    for counter, key, want in [
            ([0] * 4, [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([ones] * 4, [ones, ones], [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])]:
        assert [int(w) for w in philox(counter, key)] == want


def test_reference_masks():
    assert kept_share(0) == 65536 and kept_share(1) == 0 and kept_share(0.5) == 32768 and kept_share(2.0 ** -18) == 65536
    rows, width, p = 4000, 37, 0.3
    kept = mask(rows, width, p, 123, 5)
    # a share of n draws is off by more than six deviations hardly ever
    assert abs(kept.mean() - (1 - p)) < 6 * np.sqrt(p * (1 - p) / kept.size)
    assert not np.array_equal(kept, mask(rows, width, p, 124, 5)) and not np.array_equal(kept, mask(rows, width, p, 123, 6))
    assert np.array_equal(kept[7:], mask(rows - 7, width, p, 123, 5, first_row=7))
    assert np.array_equal(mask(2, 8, p, -1, -2), mask(2, 8, p, 2 ** 64 - 1, 2 ** 64 - 2))
    assert set(np.unique(factors(10, 10, 0.5, 1, 0))) == {0.0, 2.0} and not factors(10, 10, 1, 1, 0).any()


@pytest.mark.parametrize("call", [
    lambda x: dropout(x, 0.5, 1), lambda x: layer_norm(x), lambda x: norm_act_dropout(x, activation='relu', p=0.5),
    lambda x: rt.dropout_forward(x, 0.5, 1), lambda x: rt.layer_norm_forward(x, None, None, 1e-5),
    lambda x: rt.layer_norm_backward(x, x, x, None, None)])
def test_host_tensors_and_other_types_are_refused(call):
    for x in (torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.complex64),
              torch.zeros(3, 4).to_sparse()):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call(x)


def test_modules_check_their_arguments():
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="p has to lie"):
            Compressgnn_Dropout(p)
        with pytest.raises(ValueError, match="p has to lie"):
            Compressgnn_LayerNorm(4, p=p)
    with pytest.raises(ValueError, match="activation"):
        Compressgnn_LayerNorm(4, activation="gelu")
    with pytest.raises(ValueError, match="activation"):
        norm_act_dropout(torch.zeros(3, 4), activation="gelu")
    norm = Compressgnn_LayerNorm(4)
    for x in (torch.zeros(3, 5), torch.zeros(())):
        with pytest.raises(ValueError, match="rows of 4 features"):
            norm(x)
    assert [tuple(p.shape) for p in norm.parameters()] == [(4,), (4,)]
    assert list(Compressgnn_LayerNorm(4, affine=False).parameters()) == []
    x = torch.zeros(3, 5)
    assert Compressgnn_Dropout(0.5).eval()(x) is x and Compressgnn_Dropout(0.0)(x) is x


def test_state_dict_holds_the_place_in_the_masks():
    torch.manual_seed(3)
    a = Compressgnn_Dropout(0.5)
    b = Compressgnn_Dropout(0.5)
    assert a.seed != b.seed
    torch.manual_seed(3)
    assert Compressgnn_Dropout(0.5).seed == a.seed
    a.calls = 17
    b.load_state_dict(a.state_dict())
    assert (b.seed, b.calls) == (a.seed, 17)
    assert Compressgnn_Dropout(0.5, seed=(1 << 63) - 1).state_dict()["_extra_state"][0] == (1 << 63) - 1


def test_the_place_among_captured_calls_travels_too():
    a, b = Compressgnn_LayerNorm(4, p=0.5), Compressgnn_LayerNorm(4, p=0.5)
    a.replays.fill_(11)
    b.load_state_dict(a.state_dict())
    assert b.replays.tolist() == [11]


def test_a_module_draws_no_mask_in_a_backward_pass():
    """What is computed again there would be another function than the one whose gradient is asked for."""
    drop = Compressgnn_Dropout(0.5, seed=1)

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, grad):
            drop._next_mask(grad)
            return grad

    drop._next_mask(torch.zeros(1))
    with pytest.raises(RuntimeError, match="within a backward pass"):
        Again.apply(torch.zeros(1, requires_grad=True)).backward()
    assert drop.calls == 1


def _norm(**changed):
    call = dict(rows=4, F=8, dtype=0, param=0, ldx=8, eps=1e-5, drop=None, x=16, out=16)
    call.update(changed)
    return abi.lib().cgnn_layer_norm(abi.i64(call["rows"]), abi.i64(call["F"]), call["dtype"], call["param"], ctypes.c_void_p(call["x"]),
                                     abi.i64(call["ldx"]), None, None, ctypes.c_double(call["eps"]), 0, call["drop"],
                                     ctypes.c_void_p(call["out"]), None, None)


def _gradients(**changed):
    call = dict(rows=4, F=8, dtype=0, param=0, ldx=8, ldg=8, drop=None, x=16, grad=16, stats=16, dx=0, dw=0, ws=0, bytes=0)
    call.update(changed)
    at = ctypes.c_void_p
    return abi.lib().cgnn_layer_norm_backward(
        abi.i64(call["rows"]), abi.i64(call["F"]), call["dtype"], call["param"], at(call["grad"]), abi.i64(call["ldg"]), at(call["x"]),
        abi.i64(call["ldx"]), at(call["stats"]), None, None, 0, call["drop"], at(call["dx"]), at(call["dw"]), None, at(call["ws"]),
        ctypes.c_size_t(call["bytes"]), None)


def _dropout(**changed):
    call = dict(rows=4, F=8, dtype=0, ldx=8, x=16, out=16, drop=ctypes.byref(abi.drop_struct(0.5, 1)))
    call.update(changed)
    return abi.lib().cgnn_dropout(abi.i64(call["rows"]), abi.i64(call["F"]), call["dtype"], ctypes.c_void_p(call["x"]),
                                  abi.i64(call["ldx"]), call["drop"], ctypes.c_void_p(call["out"]), None)


def _kept(kept):
    drop = abi.drop_struct(0.5, 1)
    drop.kept = kept
    return ctypes.byref(drop)


def test_entry_points_check_before_they_touch_the_device():
    """Every call here is refused, or has nothing to do, on the host: no address in it is ever read."""
    for call in (dict(rows=-1), dict(F=-1), dict(ldx=-1), dict(ldx=7), dict(x=0), dict(out=0), dict(drop=_kept(-1)), dict(drop=_kept(65537))):
        assert _norm(**call) == EINVAL and _dropout(**call) == EINVAL, call
    assert _dropout(drop=None) == EINVAL and _norm(F=1 << 31, ldx=1 << 31) == EINVAL and _gradients(F=1 << 31, ldx=1 << 31, ldg=1 << 31, dx=16) == EINVAL
    for eps in (-1e-9, float("nan"), float("inf")):
        assert _norm(eps=eps) == EINVAL
    assert _norm(dtype=4, param=4) == EUNSUPPORTED and _dropout(dtype=-1) == EUNSUPPORTED
    for dtype, param in ((0, 1), (1, 0), (2, 3), (3, 1)):
        assert _norm(dtype=dtype, param=param) == EINVAL and _gradients(dtype=dtype, param=param, dx=16) == EINVAL
    for empty in (dict(rows=0), dict(F=0)):
        assert _norm(**empty) == 0 and _dropout(**empty) == 0
        assert _gradients(**empty) == EINVAL
    for call in (dict(ldg=-1), dict(ldx=-1), dict(ldx=7, dx=16), dict(ldg=0, dx=16), dict(x=0, dx=16), dict(grad=0, dx=16), dict(stats=0, dx=16), dict(drop=_kept(70000), dx=16)):
        assert _gradients(**call) == EINVAL, call
    assert _gradients(dtype=9, param=9) == EUNSUPPORTED
    assert _gradients() == 0  # nothing wanted
    for rows, width, dtype in ((5000, 8, 0), (5000, 8, 3), (300, 100000, 2)):
        need = abi.lib().cgnn_layer_norm_backward_workspace_bytes(abi.i64(rows), abi.i64(width), dtype)
        call = dict(rows=rows, F=width, dtype=dtype, param=dtype, ldx=width, ldg=width, dw=16)
        assert need > 0
        assert _gradients(**call) == EWORKSPACE and _gradients(**call, ws=16, bytes=need - 1) == EWORKSPACE
        assert _gradients(**call, ws=0, bytes=need) == EWORKSPACE
    assert abi.lib().cgnn_layer_norm_backward_workspace_bytes(abi.i64(0), abi.i64(8), 0) == 0
    # the graph and cluster entry points still take two types only
    assert abi.lib().cgnn_lsh_hash(abi.i64(4), abi.i64(4), 2, 2, None, None, None, None, None) != 0
