"""Device-resident autograd values, mirroring nn::Value (include/nn/autograd/value.hpp:74-228,
src/autograd/value.cpp).

A Value holds its data (a CUDA tensor used as a plain buffer) and a gradient buffer. The
gradient convention is the reference's grad_accum (value.cpp:60-64): a buffer that nothing has
written yet is "fresh", and the first backward rule that reaches it STORES its contribution;
later rules ADD. Every op's backward passes that `first` flag straight to the C ABI, so no
gradient buffer is ever zero-filled. backward() orders the graph with the reference's iterative
post-order DFS (value.cpp:80-132), seeds the root's gradient with 1 and runs the rules in reverse
topological order.

torch provides allocation and streams only; every number is produced by a kernel of libnnb.so.
"""
from __future__ import annotations

import functools
import threading
from typing import Callable, Sequence

import torch

from . import check, lib


def current_stream() -> int:
    """The current CUDA stream's handle, without building a torch.cuda.Stream around it (3 us a call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


@functools.cache
def _device(index: int) -> torch.device:
    return torch.device("cuda", index)


def empty(shape, dtype=torch.float32, device=None):
    """An uninitialised device buffer (plumbing: no kernel runs)."""
    return torch.empty(shape, dtype=dtype, device=_device(torch.cuda.current_device()) if device is None else device)


_ONES: dict = {}


def _one(device) -> torch.Tensor:
    """A device scalar 1.0 (uploaded once per device; the seed of backward())."""
    key = str(device)
    if key not in _ONES:
        _ONES[key] = torch.tensor([1.0], dtype=torch.float32, device=device)
    return _ONES[key]


class Value:
    __slots__ = ("data", "grad", "grad_fresh", "grad_borrowed", "requires_grad", "parents", "backward_fn", "name",
                 "__weakref__")

    def __init__(self, data: torch.Tensor, requires_grad: bool = False, parents: Sequence["Value"] = (),
                 backward_fn: Callable[[torch.Tensor], None] | None = None):
        self.data = data
        self.grad: torch.Tensor | None = None
        self.grad_fresh = False
        self.grad_borrowed = False           # grad is a caller's seed: read, never written
        self.requires_grad = requires_grad
        self.parents = tuple(parents)
        self.backward_fn = backward_fn
        self.name = ""

    # -- construction (value.cpp:26-45) --------------------------------------------------------
    @staticmethod
    def leaf(data: torch.Tensor, requires_grad: bool = False) -> "Value":
        v = Value(data, requires_grad)
        if requires_grad:
            v.grad = torch.empty_like(data)
            v.grad_fresh = True          # stands for zeros until the first write
        return v

    @staticmethod
    def node(data: torch.Tensor, parents: Sequence["Value"], backward_fn) -> "Value":
        if not any(p.requires_grad for p in parents):
            return Value(data, False)
        return Value(data, True, parents, backward_fn)

    # -- gradient access -----------------------------------------------------------------------
    def grad_accum(self) -> tuple[torch.Tensor, int]:
        """The gradient buffer and whether this contribution is the first (store) or not (add).

        A parameter's buffer may be a per-group view set by the data-parallel step (nnb.train); it is
        used as given."""
        if self.grad is None:
            self.grad = torch.empty_like(self.data)
            self.grad_fresh = True
        elif self.grad_borrowed:
            seed, self.grad = self.grad, torch.empty_like(self.data)
            if not self.grad_fresh:
                check(lib().nnb_accumulate(current_stream(), seed.numel(), seed.data_ptr(),
                                           self.grad.data_ptr(), 1, 0))
        self.grad_borrowed = False
        first = 1 if self.grad_fresh else 0
        self.grad_fresh = False
        return self.grad, first

    def zero_grad(self) -> None:
        """Marks the gradient as all zeros without writing it (value.cpp:69-76)."""
        if self.grad is None or self.grad.shape != self.data.shape or self.grad_borrowed:
            self.grad = torch.empty_like(self.data)
            self.grad_borrowed = False
        self.grad_fresh = True

    @property
    def shape(self):
        return tuple(self.data.shape)

    # -- backward (value.cpp:80-132) -----------------------------------------------------------
    def backward(self, seed: torch.Tensor | None = None) -> None:
        """Runs the backward rules; the root's gradient is 1, or `seed` (a device tensor with the
        root's element count: an upstream gradient, which lets a non-scalar root be differentiated
        as the reference's tests do with sum(y * g))."""
        backward((self,), (seed,))


class _Run(threading.local):
    token: object = None


_RUN = _Run()


def running() -> object:
    """A token of this thread's running backward pass: a rule that leaves something for a later rule of
    the same pass keeps the token beside it, so that what a pass that failed half-way left is not used."""
    return _RUN.token


def backward(roots: Sequence[Value], seeds: Sequence[torch.Tensor | None]) -> None:
    """Value.backward from several roots at once, each with its upstream gradient (None: 1, for a
    single-element root): the gradients of the sum over roots of sum(root * seed). A root may depend on
    another; its own seed and what reaches it through the other are added. The seeds are not written."""
    if len(roots) != len(seeds) or not roots:
        raise ValueError("backward(): needs as many seeds as roots, and at least one")
    if len({id(r) for r in roots}) != len(roots):
        raise ValueError("backward(): the same root twice")
    for root, seed in zip(roots, seeds):
        data = root.data
        if seed is None:
            if data.numel() != 1:
                raise ValueError("backward() needs a single-element value (AutogradShapeError)")
        elif seed.numel() != data.numel():
            raise ValueError("backward(): the seed must have the root's element count")
        elif seed.dtype is not data.dtype or seed.get_device() != data.get_device():
            raise ValueError("backward(): the seed must have the root's type and device")
    # iterative post-order walk over the values that have a rule (a value without one has no parents)
    topo: list[Value] = []
    done: dict[int, bool] = {}               # False: its parents are on the stack; True: in topo
    stack = list(roots)
    while stack:
        v = stack[-1]
        seen = done.get(id(v))
        if seen is None:
            done[id(v)] = False
            for p in v.parents:
                if p.backward_fn is not None and id(p) not in done:
                    stack.append(p)
            continue
        stack.pop()
        if not seen:
            done[id(v)] = True
            topo.append(v)
    seeded = {id(r) for r in roots}
    for v in topo:
        if v.backward_fn is not None and id(v) not in seeded:
            if v.grad is None or v.grad.shape != v.data.shape or v.grad_borrowed:
                v.grad = torch.empty_like(v.data)
                v.grad_borrowed = False
            v.grad_fresh = True
    for root, seed in zip(roots, seeds):
        seed = _one(root.data.device) if seed is None else seed.contiguous()
        root.grad = seed if seed.shape == root.data.shape else seed.view(root.data.shape)
        root.grad_fresh, root.grad_borrowed = False, True
    outer, _RUN.token = _RUN.token, object()
    try:
        for v in reversed(topo):
            if v.backward_fn is not None:
                v.backward_fn(v.grad)
    finally:
        _RUN.token = outer
