"""The row-wise operators as far as the host alone shows them: their sources, launches, modules.  No GPU needed."""
import copy
import glob
import os
import pickle
import re
import threading

import pytest
import torch

from compressgnn_amd import build
from CompressgnnDropout import Compressgnn_Dropout
from CompressgnnNorm import Compressgnn_LayerNorm
from launches import record
from row_shapes import CODES, many


# ------------------------------------------------------------------------- sources --
def _assembly_blocks():
    """(file, text) of every asm statement's template among the sources, pieces joined."""
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*"))):
        text = open(path).read()
        for found in re.finditer(r'\basm\s*(?:volatile\s*)?\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
            yield os.path.basename(path), "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', found[1]))


def test_wide_stores_in_assembly_keep_their_registers():
    """On gfx950 the data of a store of more than 8 bytes may not be written by the vector ALU within two wait states; the compiler does
    not see a store in assembly, so the two stand behind it in the same block (s_nop n gives n + 1)."""
    stores = 0
    for name, text in _assembly_blocks():
        steps = [step.strip() for step in re.split(r"\\n|;", text.replace("\\t", " ")) if step.strip()]
        for k, step in enumerate(steps):
            if re.match(r"(global|buffer|flat|scratch)_store_dwordx[34]\b", step):
                stores += 1
                waited = re.match(r"s_nop (\d+)$", steps[k + 1]) if k + 1 < len(steps) else None
                assert waited and int(waited[1]) + 1 >= 2, (name, text)
    assert stores


# ------------------------------------------------------------------------ launches --
def _fits(launches):
    """What HIP takes: fewer than 2^32 threads a dimension, fewer than 2^31 workgroups in the first and 2^16 in the others."""
    for kernel, grid, block in launches:
        for k in range(3):
            assert 1 <= grid[k] < (1 << 31 if k == 0 else 1 << 16) and grid[k] * block[k] < 1 << 32, (kernel, grid, block)


@pytest.mark.parametrize("dtype,width", [(3, 1 << 25), (2, (1 << 25) + 16), (0, 1 << 26), (1, 1 << 27), (3, (1 << 31) - 65537)])
def test_sums_of_wide_parameters_fit_a_launch(tmp_path, dtype, width):
    calls = [dict(op="gradients", rows=rows, F=width, dtype=dtype, relu=True, kept=30000) for rows in (1, 64, 65, 1000)]
    results, _ = record(tmp_path, calls)
    for call, (status, launches) in zip(calls, results):
        assert status == 0 and launches[0][0][0] == "norm_long_dx_kernel", call
        assert ("norm_sum_parts_kernel" in [kernel[0] for kernel, _, _ in launches]) == (call["rows"] > 64)
        _fits(launches)


@pytest.mark.parametrize("rows,width,dtype", [((1 << 33) - 512, 1, 3), (1 << 33, 1, 3), ((1 << 33) + 1000, 1, 2), ((1 << 35) + 5, 1, 0), (1 << 32, 1, 1),
                                              (1 << 33, 8, 3), ((1 << 20) + 1, 12345, 3)])
def test_dropout_of_any_number_of_rows_fits_its_launches(tmp_path, rows, width, dtype):
    (status, launches), = record(tmp_path, [dict(op="dropout", rows=rows, F=width, dtype=dtype, kept=30000)])[0]
    assert status == 0 and {kernel[0] for kernel, _, _ in launches} == {"dropout_kernel"}
    _fits(launches)
    packs = 16 // (8 if dtype == 1 else 4 if dtype == 0 else 2)
    lane = max(2, 8 // packs)  # packs that a lane takes
    whole = -(-width // 8) * (8 // packs) * rows if width % 8 else width * rows // packs
    assert sum(grid[0] for _, grid, _ in launches) == -(-whole // (256 * lane))


@pytest.mark.parametrize("rows,width,dtype", [(1 << 35, 1, 2), ((1 << 35) + 77, 1, 3), ((1 << 35) - 2048, 1, 2), (1 << 36, 1, 2), (1 << 35, 9, 3), (1 << 35, 3, 0),
                                              (1 << 29, 128, 2), (1 << 26, 1200, 3), (1 << 24, 8000, 0), (1 << 40, 1, 1)])
def test_norms_of_any_number_of_rows_fit_a_launch(tmp_path, rows, width, dtype):
    calls = [dict(op=op, rows=rows, F=width, dtype=dtype, relu=True, kept=30000) for op in ("norm", "gradients")]
    for status, launches in record(tmp_path, calls)[0]:
        assert status == 0
        _fits(launches)


@pytest.mark.parametrize("dtype", range(4))
def test_parts_keep_a_lanes_chain_short(tmp_path, dtype):
    """The parameters' sums are added in float down the rows of a part and in 64 bits from part to part: no lane adds more than 1,024 rows."""
    calls = [dict(op="gradients", rows=rows, F=width, dtype=dtype) for width in (1, 40, 1000, 8193, 20001)
             for rows in (5, 1000, 100003, (1 << 21) + 5, 1 << 24, (1 << 28) - 1) if rows * width < 1 << 38]
    for call, (status, launches) in zip(calls, record(tmp_path, calls)[0]):
        assert status == 0
        _fits(launches)
        for (name, values), grid, block in launches:
            if name == "norm_gradients_kernel":
                assert -(-call["rows"] // (grid[0] * (block[0] // values[1]))) <= 1024, call
            if name == "norm_long_parts_kernel":
                assert -(-call["rows"] // grid[1]) <= 4 * 1024, call


# ------------------------------------------------------------------------- modules --
@pytest.mark.parametrize("module", [Compressgnn_Dropout(0.5, seed=1), Compressgnn_LayerNorm(4, p=0.5, seed=1)])
def test_a_module_draws_no_mask_under_a_trace(module):
    """The number of the call would be a constant of the trace, and every run of it drop the same elements."""
    class Masked(torch.nn.Module):
        def forward(self, x):
            return x * float(module._next_mask(x)[1])

    with pytest.raises(RuntimeError, match="a trace would draw"):
        torch.jit.trace(Masked(), (torch.ones(3, 4),), check_trace=False)
    assert module.calls == 0
    # in eval mode nothing is drawn, and a trace of the whole module holds what it computes
    drop = Compressgnn_Dropout(0.5).eval()
    x = torch.ones(3, 4)
    assert torch.equal(torch.jit.trace(drop, (x,), check_trace=False)(x * 2), x * 2)


def test_deep_copies_draw_masks_of_their_own():
    """As layers are stacked: one is made and copied, and no two of them may drop the same elements."""
    layer = torch.nn.Sequential(torch.nn.Linear(4, 4), Compressgnn_LayerNorm(4, activation="relu", p=0.5, seed=5), Compressgnn_Dropout(0.3))
    layer[1].weight.data.fill_(2.0)
    layer[1].calls, layer[1].tied = 7, layer[1].weight
    layer[1].replays.fill_(3)
    before = layer[1].seed
    stack = [copy.deepcopy(layer) for _ in range(6)] + [layer]
    assert layer[1].seed == before
    for k in (1, 2):
        assert len({layers[k].seed for layers in stack}) == len(stack)
    for layers in stack[:-1]:
        norm = layers[1]
        assert type(norm) is Compressgnn_LayerNorm and norm.p == 0.5 and norm.activation == "relu" and norm.calls == 7
        assert torch.equal(norm.weight, layer[1].weight) and norm.weight is not layer[1].weight and norm.tied is norm.weight
        assert isinstance(norm.weight, torch.nn.Parameter) and norm.replays.tolist() == [3] and norm.replays is not layer[1].replays
        assert [name for name, _ in layers.named_parameters()] == [name for name, _ in layer.named_parameters()]
    torch.manual_seed(11)
    seeds = [copy.deepcopy(layer[2]).seed for _ in range(2)]
    torch.manual_seed(11)
    assert [copy.deepcopy(layer[2]).seed for _ in range(2)] == seeds and seeds[0] != seeds[1]
    twice = copy.deepcopy([layer[2], layer[2]])  # one module twice stays one
    assert twice[0] is twice[1]
    # the state dict and a pickle carry the place in the masks
    other = copy.deepcopy(layer)
    other.load_state_dict(layer.state_dict())
    assert (other[1].seed, other[1].calls) == (before, 7) and other[2].seed == layer[2].seed
    same = pickle.loads(pickle.dumps(layer))
    assert (same[1].seed, same[1].calls, same[2].seed) == (before, 7, layer[2].seed)


def test_modules_are_made_on_the_device_without_memory():
    """As large models are laid out before their weights are there."""
    with torch.device("meta"):
        layers = torch.nn.Sequential(Compressgnn_LayerNorm(4, p=0.5), Compressgnn_Dropout(0.5))
        stack = [copy.deepcopy(layers) for _ in range(2)]
    assert layers[0].weight.is_meta and layers[1].replays.is_meta
    assert len({module.seed for layers in [layers, *stack] for module in layers}) == 6
    torch.manual_seed(3)
    seed = Compressgnn_Dropout(0.5).seed
    torch.manual_seed(3)
    with torch.device("meta"):
        assert Compressgnn_Dropout(0.5).seed == seed


def test_calls_from_two_threads_get_two_numbers():
    """A second call that comes while the first is between reading the count and writing it: forced, not hoped for."""
    numbers = {}

    class Slow(Compressgnn_Dropout):
        @property
        def calls(self):
            return self.__dict__["_calls"]

        @calls.setter
        def calls(self, value):
            self.__dict__["_calls"] = value
            if value == 1 and "second" not in numbers:
                numbers["second"] = None
                late.start()
                late.join(0.5)  # where calls wait for each other it comes to nothing before this one is through

    module = Slow(0.5, seed=3)
    x = torch.zeros(2, 2)
    late = threading.Thread(target=lambda: numbers.update(second=module._next_mask(x)[1]))
    first = module._next_mask(x)[1]
    late.join(30)
    assert sorted([first, numbers["second"]]) == [0, 1] and module.calls == 2


def test_state_dicts_of_torchs_modules_are_loaded():
    """A model that had torch's LayerNorm and Dropout in these places: its parameters are there, a place in masks is not."""
    theirs = torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.LayerNorm(4), torch.nn.Dropout(0.5))
    torch.nn.init.normal_(theirs[1].weight)
    for p in (0.0, 0.5):
        ours = torch.nn.Sequential(torch.nn.Linear(3, 4), Compressgnn_LayerNorm(4, p=p, seed=5), Compressgnn_Dropout(0.5, seed=6))
        ours[1].calls = 2
        ours[2].replays.fill_(4)
        done = ours.load_state_dict(theirs.state_dict())
        assert not done.missing_keys and not done.unexpected_keys
        assert torch.equal(ours[1].weight, theirs[1].weight) and torch.equal(ours[1].bias, theirs[1].bias)
        assert (ours[1].seed, ours[1].calls, ours[2].seed, ours[2].replays.tolist()) == (5, 2, 6, [4])
    # half a place, and a parameter that is not there, are still missed
    for k, lost in ((1, "1.replays"), (1, "1._extra_state"), (2, "2.replays"), (1, "1.weight"), (1, "1.bias")):
        state = ours.state_dict()
        del state[lost]
        with pytest.raises(RuntimeError, match=re.escape(lost)):
            ours.load_state_dict(state)
        assert ours.load_state_dict(state, strict=False).missing_keys == [lost]
    state = theirs.state_dict()
    del state["1.bias"]
    with pytest.raises(RuntimeError, match="1.bias"):
        ours.load_state_dict(state)
    with pytest.raises(RuntimeError, match="Unexpected"):
        ours.load_state_dict(dict(theirs.state_dict(), **{"1.more": torch.zeros(1)}))


# -------------------------------------------------------------------------- shapes --
def test_no_sum_of_parts_is_built_that_no_call_takes(tmp_path):
    calls = [dict(op="gradients", rows=100000, F=64, dtype=dtype, param=param) for dtype, param in ((0, 0), (1, 1), (2, 2), (2, 0), (3, 3), (3, 0))]
    results, kernels = record(tmp_path, calls)
    reached = {kernel for _, launches in results for kernel, _, _ in launches}
    built = {kernel for kernel in kernels if kernel[0] == "norm_sum_parts_kernel"}
    assert built <= reached, built - reached


def test_every_kernel_of_the_norm_is_reached_by_the_tests_with_formulas(tmp_path):
    """Each instance of the row kernels that the library has, type by type, ReLU and dropout in all four ways, is what one of the matrices
    launches that are compared with the formulas in 64 bits on the GPU."""
    from test_gpu_norm import SHAPES
    calls, wanted = [], []
    for dtype, code in CODES.items():
        for param in {code, 0} if code > 1 else {code}:
            for relu, kept in ((False, None), (True, None), (False, 45875), (True, 32768)):
                for shape, (rows, width) in [(None, s) for s in SHAPES] + [(shape, (rows, width)) for shape, rows, width in many(dtype)]:
                    for op in ("norm", "gradients"):
                        calls.append(dict(op=op, rows=rows, F=width, dtype=code, param=param, relu=relu, kept=kept))
                        wanted.append(shape if op == "norm" else None)
    results, kernels = record(tmp_path, calls)
    reached = set()
    for call, shape, (status, launches) in zip(calls, wanted, results):
        assert status == 0
        reached.update(kernel for kernel, _, _ in launches)
        if shape:
            (name, values), = [kernel for kernel, _, _ in launches]
            assert name == "norm_rows_kernel" and values[1:3] == shape, (call, name, values, shape)
    missing = [kernel for kernel in kernels if kernel[0].startswith("norm_") and kernel not in reached]
    assert not missing, sorted(missing)
    assert sum(kernel[0] == "norm_rows_kernel" for kernel in reached) > 4 * 4 * 18


@pytest.mark.parametrize("dtype", [2, 3])
@pytest.mark.parametrize("rows,param,packs", [(2048, 0, 1), (4096, 0, 1), (4097, 0, 2), (2048, 2, 1), (3584, 2, 1), (3585, 2, 2), (4096, 2, 2)])
def test_wide_16_bit_rows_are_spread_where_that_was_faster(tmp_path, dtype, rows, param, packs):
    """4,096 features: a pack a lane under float32 parameters up to 4,096 rows, under parameters of the rows' type only where it gained."""
    (_, launches), = record(tmp_path, [dict(op="norm", rows=rows, F=4096, dtype=dtype, param=dtype if param == 2 else 0)])[0]
    (name, values), = [kernel for kernel, _, _ in launches]
    assert name == "norm_rows_kernel" and values[1:3] == ((512, 1) if packs == 1 else (256, 2))
