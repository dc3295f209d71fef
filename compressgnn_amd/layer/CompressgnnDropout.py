"""Dropout of node features whose mask is never stored: out = x / (1 - p) where an element is kept, else 0.

The reference's models take dropout from torch; here it is a kernel that finds the mask from (seed, offset) and the
position of an element, in the forward pass and again in the gradient.  The share of kept elements is taken to the
nearest 65,536th and the scale is its reciprocal.  Rows are the last dimension; the mask of an element depends on its row and
its column, not on the type or on strides.
"""
import copy
import threading

import _paths  # noqa: F401
import torch
from torch.autograd.function import once_differentiable

import compressgnn_runtime as _native


class _Dropped(torch.autograd.Function):
    """(x, p, seed, offset, counter) -> out: the step of _native.dropout, for what a native one does not take part in"""

    @staticmethod
    def forward(ctx, x, p, seed, offset, counter):
        ctx.save_for_backward(counter)
        ctx.mask = (p, seed, offset)
        return _native.dropout_forward(x, p, seed, offset, counter)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (counter,) = ctx.saved_tensors
        return _native.dropout_forward(grad, *ctx.mask, counter), None, None, None, None


def dropout(x, p, seed, offset=0, counter=None):
    """x with elements dropped with probability p, the others scaled by 1 / (1 - p); a dropped element is 0 whatever it holds.

    seed, offset: whole numbers that name the mask; equal ones give equal masks.  counter: an int64 tensor of one
    element beside x that is added to offset when the kernel runs; it must not be written to between a call and its
    gradient (autograd refuses that).  A step captured into a graph that counts it up draws another mask in each replay."""
    out = _native.dropout(x, p, seed, offset, counter)
    return _Dropped.apply(x, p, seed, offset, counter) if out is None else out


def _fresh_seed():
    """Of torch's own generator, where none is given: torch.manual_seed fixes it, and no two modules share masks."""
    return int(torch.randint(1 << 62, (1,), device="cpu"))  # whatever device modules are being made on, the one without memory too


_numbering = threading.Lock()  # no two calls get one number, whatever threads they come from


class Masks:
    """The masks of a module, one after the other: each is named by the module's seed and the number of the call.

    Calls under a stream capture are numbered on the device, by a counter that the captured work itself
    counts up, and lie in a range of their own; the module has to be on the device of the rows before.  A deep copy of a
    module, as layers are stacked with, is a module of its own and gets a seed of its own, of torch's generator; the state dict carries the
    seed and the place from one module to another.  A forward pass computed again in a backward one (activation checkpointing) would draw
    other masks than the first time and is refused, and so is one under a trace (torch.jit.trace), which would hold one call's number and
    drop the same elements in every run: there the functions, whose masks have names, serve."""

    CAPTURED = 1 << 62  # offsets of captured calls begin here

    def _init_masks(self, seed):
        self.seed = _fresh_seed() if seed is None else int(seed)
        self.calls = 0
        self.register_buffer('replays', torch.zeros(1, dtype=torch.int64))

    def __deepcopy__(self, memo):
        twin = type(self).__new__(type(self))
        memo[id(self)] = twin
        twin.__dict__.update(copy.deepcopy(self.__dict__, memo))
        twin.seed = _fresh_seed()
        return twin

    def _next_mask(self, x):
        """(seed, offset, counter) of a call on x"""
        if _native.in_backward():
            raise RuntimeError("a call within a backward pass would draw another mask than the forward pass did; call dropout or "
                               "norm_act_dropout with a seed and an offset where activations are computed again")
        if torch.jit.is_tracing():
            raise RuntimeError("a trace would draw the mask of this one call in every run; trace the module in eval mode, or call dropout or "
                               "norm_act_dropout with a seed, an offset and a counter on the device")
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            if self.replays.device != x.device:
                raise RuntimeError("the module is on %s and x on %s: move it there before the capture" % (self.replays.device, x.device))
            counter = self.replays + 0
            self.replays += 1
            return self.seed, self.CAPTURED, counter
        with _numbering:
            number = self.calls
            self.calls = number + 1
        return self.seed, number, None

    def get_extra_state(self):
        return torch.tensor([self.seed, self.calls], dtype=torch.int64)

    def set_extra_state(self, state):
        self.seed, self.calls = (int(v) for v in state)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        """A state dict without a place in the masks at all is that of a model with torch's modules: the place stays as it is."""
        missing = []
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing, unexpected_keys, error_msgs)
        place = {prefix + "replays", prefix + "_extra_state"}
        missing_keys += [key for key in missing if key not in place or any(part in state_dict for part in place)]


class Compressgnn_Dropout(Masks, torch.nn.Module):
    """dropout(x, p) in training, x itself otherwise.  seed: fixes the masks; its own and the numbers of calls so far, captured
    ones too, travel with the state dict, so that training resumed from one draws the masks it would have drawn."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError("p has to lie in [0, 1], got %r" % (p,))
        self.p = p
        self._init_masks(seed)

    def forward(self, x):
        if not self.training or self.p == 0:
            return x
        return dropout(x, self.p, *self._next_mask(x))

    def extra_repr(self):
        return "p=%g" % self.p
