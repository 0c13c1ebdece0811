"""What the training operators' direct entry points share: argument checks, and calls kept by layout.

An entry point validates a call, chooses its launches and describes them as a `Plan`: the buffers to
allocate, results first, and per launch a kernel, its grid and its arguments, in which `tensor(i)` stands
for the call's i-th tensor and `buffer(j)` for the j-th buffer.  A `Table` keeps plans by everything that
validation and launch choice read (the tensors' dtypes, devices, sizes, strides and 16-byte alignment, and
the call's numbers), so that a layout seen before costs one lookup, the allocations and the launches, in
C++ (CallTable in csrc/nep_dispatch.cpp).  A plan holds metadata only.
"""
from __future__ import annotations

from neptune_codegen import dispatch, hip

# a launch has fewer than 2^32 work-items in each dimension of its grid
MOST_THREADS = (1 << 32) - 1
# what kernels take as an fp32 number, and as its product with a number below 4
LEAST_FLOAT, MOST_FLOAT = 2.0 ** -126, 2.0 ** 125


class tensor:
    """Kernel argument: the address of the call's tensor `index` (null where that is None)."""

    __slots__ = ("index",)

    def __init__(self, index: int):
        self.index = index


class buffer:
    """Kernel argument: the address of buffer `index` and `add` bytes."""

    __slots__ = ("index", "add")

    def __init__(self, index: int, add: int = 0):
        self.index, self.add = index, add


class Plan:
    """One call layout.  `buffers`: (shape, dtype), results and scratch; `returns`: the buffer of each
    result, None for an absent one; `bare`: a single result comes without a tuple."""

    def __init__(self, device: int, n_tensors: int, buffers, returns, launches, bare: bool = False):
        self.device, self.buffers, self.returns, self.bare = device, tuple(buffers), tuple(returns), bare
        self.launches = tuple(launches)
        native = []
        for kernel, grid, args in self.launches:
            plain = tuple(0 if isinstance(a, (tensor, buffer)) else a for a in args)
            if len(plain) != len(kernel.argtypes):
                raise TypeError(f"{kernel.name}: expected {len(kernel.argtypes)} arguments, got {len(plain)}")
            patches = tuple((kernel.pointer_offsets[i], a.index if isinstance(a, tensor) else -1 - a.index,
                             0 if isinstance(a, tensor) else a.add)
                            for i, a in enumerate(args) if isinstance(a, (tensor, buffer)))
            check_grid(grid, kernel.block, kernel.name)
            native.append((kernel.handle, (*grid, 1, 1)[:3], kernel.block, kernel.lds,
                           kernel._packer.pack(*plain), patches))
        code = {}
        for _, dtype in self.buffers:
            code[dtype] = _dtype_code(dtype)
        self.native = dispatch.extension().CallPlan(
            n_tensors, tuple((code[dtype], tuple(shape)) for shape, dtype in self.buffers),
            [-1 if r is None else r for r in self.returns], bare, tuple(native))

    def run(self, tensors: tuple):
        """The results of the plan's launches on the current stream of its device."""
        if hip.recording_active():
            return self._run_recorded(tensors)
        return self.native.run(tensors)

    def _run_recorded(self, tensors):
        # through Kernel.launch, which the recorder sees
        import torch

        device = torch.device("cuda", self.device)
        out = [torch.empty(shape, dtype=dtype, device=device) for shape, dtype in self.buffers]
        for index, t in enumerate(out):
            if index not in self.returns:
                hip.scratch(t)

        def value(a):
            if isinstance(a, tensor):
                t = tensors[a.index]
                return 0 if t is None else t.data_ptr()
            return out[a.index].data_ptr() + a.add if isinstance(a, buffer) else a

        with torch.cuda.device(device):
            for kernel, grid, args in self.launches:
                kernel.launch(grid, tuple(map(value, args)), hip.current_stream(device))
        results = tuple(None if r is None else out[r] for r in self.returns)
        return results[0] if self.bare else results


_CODES: dict = {}


def _dtype_code(dtype) -> int:
    import torch

    if dtype not in _CODES:
        _CODES[dtype] = dispatch.extension().dtype_code(torch.empty(0, dtype=dtype))
    return _CODES[dtype]


class Table:
    """Plans of one entry point by call layout."""

    def __init__(self):
        self._native = None

    def native(self):
        if self._native is None:
            self._native = dispatch.extension().CallTable()
        return self._native

    def run(self, tensors: tuple, numbers: tuple):
        """The results of a call whose layout is known, or None."""
        if self._native is None or hip.recording_active():
            return None
        return self._native.run(tensors, numbers)

    def keep(self, tensors: tuple, numbers: tuple, plan: Plan) -> None:
        self.native().keep(tensors, numbers, plan.native)


def is_metadata(t) -> bool:
    from torch._subclasses.fake_tensor import FakeTensor

    return isinstance(t, FakeTensor) or t.device.type == "meta"


def device_index(t) -> int:
    import torch

    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def same(given: tuple, used: tuple) -> bool:
    """Whether a call uses its tensors as they were given (a plan with copies is not kept)."""
    return all(a is b for a, b in zip(given, used))


def rows_of(t):
    """`t` itself where its rows have one stride and unit column stride, else a contiguous copy; and the
    row stride in elements (0 of a tensor with one row)."""
    shape, strides = t.shape, t.stride()
    step, rows = None, 1
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != step * rows:
            step = -1
            break
        rows *= size
    if step == -1 or (shape[-1] > 1 and strides[-1] != 1):
        t = t.contiguous()
        step = shape[-1]
    return t, step or 0


def check_tensor(t, name: str, *, metadata: bool) -> None:
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.layout != torch.strided:
        raise TypeError(f"{name} must be strided")
    if not metadata and t.device.type != "cuda":
        raise ValueError(f"{name} is on {t.device}; execution requires a ROCm (cuda) device")


def check_grid(grid, threads: int, name: str) -> None:
    if grid[0] * threads > MOST_THREADS or any(n > 65535 for n in grid[1:]):
        raise NotImplementedError(f"{name}: the call needs a grid of {tuple(grid)} workgroups of {threads} "
                                  "threads, more than one launch takes")
