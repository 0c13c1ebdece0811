"""Embedding lookup with a scale, and the table's gradient.

There is no reference function for this path:

    out[i] = scale * table[token i]          dtable[v] = scale * sum over i with token i = v of grad[i]

Layout contract: tokens [...] in int32 or int64, a table [vocab, n] in float32, bfloat16 or float16, the
output [..., n] in its dtype.  A negative token stands for none: a row of zeros, and no gradient.  A token of
vocab or more has a row of NaN and no gradient; it is never read through.  The arithmetic is fp32 with one
rounding; the gradient's rows are added in the order of their positions, without atomics.  Formulas and
mapping are in csrc/kernels/nep_embedding.h.
"""
from __future__ import annotations

import threading

from neptune_codegen import calls, dispatch, hip
from neptune_codegen.emitters import (BASE_OPTIONS, EmbeddingVariant, embedding_few_name, embedding_order_name,
                                      embedding_sums_name, emit_embedding_few_source,
                                      emit_embedding_order_source, emit_embedding_source,
                                      emit_embedding_sums_source)

FEW = 512                # tokens that one launch takes (nep_embedding.h kFewTokens)
MOST_TOKENS = 1 << 26    # of a gradient: sixteen wavefronts' runs of 2^22
MOST_ROWS = 1 << 24      # (each thousand rows have a workgroup that reads all tokens)
MOST_KEYS = 1024         # rows that a workgroup counts the tokens of (nep_embedding.h kMostKeys)
MOST_ROW = 65535 << 10   # bytes, of more than FEW tokens' gradient (the join's grid: 65535 times 64 words)
MOST_STRIDE = 16         # of a gradient's tokens (nep_embedding.h kMostTokenStride)
_PROGRAMS: dict = {}
_OPS: dict = {}
_FORWARD, _BACKWARD = calls.Table(), calls.Table()
_lock = threading.Lock()

_LOOKUP_ARGS = (hip.PTR,) * 3 + (hip.I64, hip.I32) + (hip.I64,) * 3 + (hip.F32,)
_ORDER_ARGS = (hip.PTR,) * 4 + (hip.I64,) * 3 + (hip.I32,)
_SUMS_ARGS = (hip.PTR,) * 6 + (hip.I64, hip.I32) + (hip.I64,) * 3 + (hip.I32,) * 5 + (hip.F32,)
_FEW_ARGS = (hip.PTR,) * 3 + (hip.I32,) * 2 + (hip.I64,) * 4 + (hip.I32,) * 4 + (hip.F32,)
_JOIN_ARGS = (hip.PTR,) * 3 + (hip.I64, hip.I32) + (hip.I64,) * 2 + (hip.I32,) * 2 + (hip.F32,)


def _program(name: str, emit, *args) -> hip.Program:
    with _lock:
        prog = _PROGRAMS.get(name)
        if prog is None:
            prog = _PROGRAMS[name] = hip.Program(emit(*args), f"{name}.hip", BASE_OPTIONS)
        return prog


def _lookup_program(var: EmbeddingVariant) -> hip.Program:
    return _program(var.name, emit_embedding_source, var)


def _order_program(index: str, waves: int) -> hip.Program:
    return _program(embedding_order_name(index, waves), emit_embedding_order_source, index, waves)


def _sums_program(dtype, out, access: str, add: bool) -> hip.Program:
    return _program(embedding_sums_name("sums", dtype, out, access, add), emit_embedding_sums_source, dtype, out,
                    access, add)


def _few_program(dtype, out, index: str, access: str, add: bool) -> hip.Program:
    return _program(embedding_few_name(dtype, out, index, access, add), emit_embedding_few_source, dtype, out, index,
                    access, add)


def _scale(scale) -> float:
    if type(scale) not in (int, float) or not abs(scale) <= calls.MOST_FLOAT:
        raise ValueError("embedding needs a scale that is finite in fp32")
    return float(scale)


def _check_rows(t, name: str, *, metadata: bool) -> None:
    import torch

    calls.check_tensor(t, f"embedding {name}", metadata=metadata)
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"embedding takes float32, bfloat16 and float16, got {t.dtype} for {name}")


def _check_tokens(tokens, device, *, metadata: bool) -> None:
    import torch

    calls.check_tensor(tokens, "embedding tokens", metadata=metadata)
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.device != device:
        raise ValueError("embedding tensors must be on the same device")


def _check_sizes(tokens, vocab: int, n: int) -> None:
    if tokens.numel() >= 1 << 31 or vocab >= 1 << 31 or n >= 1 << 28:
        raise NotImplementedError("embedding takes less than 2^31 tokens and rows, and rows of less than 2^28")


def _check_gradient_sizes(tokens, vocab: int, n: int, size: int) -> None:
    if tokens.numel() >= MOST_TOKENS or vocab > MOST_ROWS:
        raise NotImplementedError("embedding's gradient takes less than 2^26 tokens, and up to 2^24 rows")
    if n * size > MOST_ROW and tokens.numel() > FEW:
        raise NotImplementedError(f"embedding's gradient of more than {FEW} tokens takes rows of up to {MOST_ROW} bytes")


def validate_embedding_inputs(tokens, table, *, metadata: bool = False) -> None:
    _check_rows(table, "table", metadata=metadata)
    if table.ndim != 2 or not table.numel():
        raise ValueError(f"embedding table must be [vocab, n] with both at least 1, got {tuple(table.shape)}")
    _check_tokens(tokens, table.device, metadata=metadata)
    _check_sizes(tokens, *table.shape)


def validate_embedding_gradient_inputs(grad, tokens, vocab, into=None, *, metadata: bool = False) -> None:
    import torch

    _check_rows(grad, "grad", metadata=metadata)
    _check_tokens(tokens, grad.device, metadata=metadata)
    if type(vocab) is not int or vocab < 1:
        raise ValueError("embedding needs a vocab of at least 1")
    if not grad.ndim or grad.shape[:-1] != tokens.shape or not grad.shape[-1]:
        raise ValueError(f"embedding grad {tuple(grad.shape)} must be [..., n] with tokens of the leading sizes, "
                         f"got {tuple(tokens.shape)}")
    n = grad.shape[-1]
    _check_sizes(tokens, vocab, n)
    _check_gradient_sizes(tokens, vocab, n, grad.element_size())
    if into is None:
        return
    calls.check_tensor(into, "embedding into", metadata=metadata)
    if into.shape != (vocab, n) or into.device != grad.device:
        raise ValueError(f"embedding into must be [{vocab}, {n}] on the gradient's device, got {tuple(into.shape)}")
    if into.dtype not in (grad.dtype, torch.float32):
        raise TypeError(f"embedding into must be float32 or {grad.dtype}, got {into.dtype}")
    if into.requires_grad:
        raise ValueError("embedding into is written in place and must not require grad")
    if (n > 1 and into.stride(1) != 1) or (vocab > 1 and into.stride(0) < n):
        raise ValueError("embedding into must have unit column stride and rows that do not overlap")


def _apart(into, *read) -> bool:
    """Whether `into` overlaps nothing that is read (what is no tensor or has no memory is refused elsewhere)."""
    import torch

    def real(t):
        return not t.is_meta if type(t) is torch.Tensor else isinstance(t, torch.Tensor) and not calls.is_metadata(t)

    return not real(into) or not any(real(t) and calls.overlap(t, into) for t in read)


def _access(n: int, *tensors) -> str:
    """`tensors`: (tensor, row stride)."""
    vec = 16 // tensors[0][0].element_size()
    if n < vec:
        return "few"
    return "words" if n % vec == 0 and all(t.data_ptr() % 16 == 0 and s % (16 // t.element_size()) == 0
                                           for t, s in tensors) else "any"


def _name(t) -> str:
    return str(t.dtype).replace("torch.", "")


def _flat(tokens, most: int | None = None):
    """Tokens whose elements have one stride (of up to `most`), and that stride."""
    used, stride = calls.rows_of(tokens.unsqueeze(-1))
    if most is not None and stride > most:
        used, stride = used.contiguous(), 1
    return (tokens if used.data_ptr() == tokens.data_ptr() else used), stride


def _lookup_variant(table, tokens, access: str, n: int) -> EmbeddingVariant:
    slots = -(-n // (16 // table.element_size()))
    tpr = min(256, 1 << max(0, (slots - 1).bit_length()))
    return EmbeddingVariant(_name(table), _name(tokens), access, tpr, 2 if slots >= 512 else 1)


def run_embedding(tokens, table, *, scale: float = 1.0):
    """Rows [..., n] of the table for tokens [...], times `scale`, in the table's dtype, on the current
    stream.  A call whose tensor layouts and scale were seen before reuses that call's kernel and launch
    shape."""
    import torch

    given = (tokens, table)
    found = _FORWARD.run(given, (scale,))
    if found is not None:
        return found
    metadata = isinstance(table, torch.Tensor) and calls.is_metadata(table)
    validate_embedding_inputs(*given, metadata=metadata)
    number, scale = scale, _scale(scale)
    (vocab, n), rows = table.shape, tokens.numel()
    shape = (*tokens.shape, n)
    if metadata or rows == 0:
        return torch.empty(shape, dtype=table.dtype, device=table.device)
    (flat, si), (used, st) = _flat(tokens), calls.rows_of(table)
    var = _lookup_variant(table, tokens, _access(n, (used, st)), n)
    slots = -(-n // (16 // table.element_size()))
    device = calls.device_index(table)
    kernel = _lookup_program(var).kernel(var.name, _LOOKUP_ARGS, 256, device)
    launch = (kernel, (-(-rows // (256 // var.tpr)), min(65535, -(-slots // (var.tpr * var.unroll)))),
              (calls.tensor(0), calls.tensor(1), calls.buffer(0), rows, n, vocab, si, st, scale))
    plan = calls.Plan(device, 2, [(shape, table.dtype)], (0,), [launch], bare=True)
    if calls.same(given, (flat, used)):
        _FORWARD.keep(given, (number,), plan)
    return plan.run((flat, used))


def _shares(vocab: int) -> int:
    """Workgroups (log 2) that the rows of the table are dealt to for the tokens' order: one a CU, or a row
    each; more where their counters would not hold the rows."""
    log = min(8, (vocab - 1).bit_length())
    while -(-vocab >> log) > MOST_KEYS:
        log += 1
    return log


def _chunk(count: int, words: int) -> int:
    """Sorted entries that a wavefront adds."""
    chunk = 16
    while chunk < 256 and -(-count // (2 * chunk)) * -(-words // 64) > 1536:
        chunk *= 2
    return chunk


def _ordered(given, table, buffers, device, access, add, out, si, sg, st, scale, vocab, chunk, columns, clear,
             log_lanes, log_tiles):
    """Launches of a gradient with more than a few tokens; adds their scratch to the buffers."""
    import torch

    grad, tokens, _ = given
    n, count, index = grad.shape[-1], tokens.numel(), _name(tokens)
    log, waves, chunks = _shares(vocab), 16 if count > 1024 else 4, -(-count // chunk)
    # keys, positions and the rows that are named; parts of runs over several chunks
    keys, positions, named, parts = (calls.buffer(len(buffers) + i) for i in range(4))
    buffers += [((count,), torch.int32)] * 2 + [((vocab,), torch.uint8)]
    buffers.append(((chunks * 2 * 64 * columns * (16 // grad.element_size()),), torch.float32))
    tag = (_name(grad), str(out), access, add)
    prog = _sums_program(*tag)
    launches = [(_order_program(index, waves).kernel(embedding_order_name(index, waves), _ORDER_ARGS, 64 * waves, device),
                 (1 << log,), (calls.tensor(1), keys, positions, named, count, vocab, si, log)),
                (prog.kernel(embedding_sums_name("sums", *tag), _SUMS_ARGS, 64, device), (chunks * columns + clear,),
                 (calls.tensor(0), keys, positions, named, table, parts, count, n, vocab, sg, st, chunk, columns,
                  chunks * columns, log_lanes, log_tiles, scale))]
    if chunks > 1:
        launches.append((prog.kernel(embedding_sums_name("join", *tag), _JOIN_ARGS, 256, device), (chunks, columns),
                         (keys, parts, table, count, n, vocab, st, chunk, chunks, scale)))
    return launches


def run_embedding_backward(grad, tokens, vocab: int, *, scale: float = 1.0, into=None):
    """Gradient [vocab, n] of the table for the output's gradient `grad` [..., n], in its dtype; or, with
    `into` [vocab, n] in that dtype or float32, the gradient added to `into` in place (one rounding for each
    row that a token names, the others untouched), and `into`, which overlaps nothing that the call reads."""
    import torch

    given, add = (grad, tokens, into), into is not None
    # (what the layout of the tensors does not say; refused below)
    apart = not add or (isinstance(into, torch.Tensor) and not into.requires_grad and _apart(into, grad, tokens))
    found = _BACKWARD.run(given, (vocab, scale)) if apart else None
    if found is not None:
        if not add:
            return found[0]
        calls.written(into)
        return into
    metadata = isinstance(grad, torch.Tensor) and calls.is_metadata(grad)
    validate_embedding_gradient_inputs(grad, tokens, vocab, into, metadata=metadata)
    if not metadata and not apart:
        raise ValueError("embedding into must not overlap the gradient that is added to it, or the tokens")
    number, scale = scale, _scale(scale)
    n, count = grad.shape[-1], tokens.numel()
    if metadata or count == 0:
        return torch.zeros((vocab, n), dtype=grad.dtype, device=grad.device) if into is None else into
    (g, sg), (flat, si) = calls.rows_of(grad), _flat(tokens, MOST_STRIDE)
    used, device = (g, flat, into), calls.device_index(grad)
    st = n if into is None else into.stride(0) if vocab > 1 else n
    out = grad.dtype if into is None else into.dtype
    words = -(-n // (16 // grad.element_size()))
    access = _access(n, (g, sg), *([(into, st)] if add else []))
    columns = -(-words // 64)
    # wavefronts that clear: four words a lane, of several short rows or a part of a long one
    log_lanes, log_tiles = min(7, (words - 1).bit_length()), (-(-words // 256) - 1).bit_length()
    clear = 0 if add else -(-vocab // (4 * (64 >> log_lanes))) if log_lanes < 7 else vocab << log_tiles
    buffers = [] if add else [((vocab, n), out)]
    table = calls.tensor(2) if add else calls.buffer(0)
    if count <= FEW:
        few = (_name(grad), str(out), _name(tokens), access, add)
        launches = [(_few_program(*few).kernel(embedding_few_name(*few), _FEW_ARGS, 256, device),
                     (count * columns + -(-clear // 4),),
                     (calls.tensor(1), calls.tensor(0), table, count, n, vocab, si, sg, st, columns, count * columns,
                      log_lanes, log_tiles, scale))]
    else:
        chunk = _chunk(count, words)
        launches = _ordered(given, table, buffers, device, access, add, out, si, sg, st, scale, vocab, chunk, columns,
                            clear, log_lanes, log_tiles)
    plan = calls.Plan(device, 3, buffers, () if add else (0,), launches)
    if calls.same(given, used):
        _BACKWARD.keep(given, (vocab, number), plan)
    made = plan.run(used)
    if add:
        calls.written(into)
        return into
    return made[0]


@dispatch.one_at_a_time
def as_embedding_op(scale: float = 1.0, lib: str = "neptune"):
    """Differentiable custom op `(Tensor tokens, Tensor table) -> Tensor` with the scale in its name; the
    gradient is the table's, and a call that it would refuse is refused before anything runs, whether or not the table
    requires grad (run_embedding takes larger tables and more tokens)."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    scale = _scale(scale)
    key = (lib, scale)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"embedding{parameter_tag({'scale': scale})}"

    def _forward(tokens, table):
        if table.ndim == 2:
            _check_gradient_sizes(tokens, *table.shape, table.element_size())
        return run_embedding(tokens, table, scale=scale)

    def _forward_fake(tokens, table):
        validate_embedding_inputs(tokens, table, metadata=True)
        _check_gradient_sizes(tokens, *table.shape, table.element_size())
        return torch.empty((*tokens.shape, table.shape[1]), dtype=table.dtype, device=table.device)

    def _backward(grad, tokens, vocab):
        return run_embedding_backward(grad, tokens, vocab, scale=scale)

    def _backward_fake(grad, tokens, vocab):
        return torch.empty((vocab, grad.shape[-1]), dtype=grad.dtype, device=grad.device)

    define = torch.library.custom_op
    op = define(f"{lib}::{name}", mutates_args=(), schema="(Tensor tokens, Tensor table) -> Tensor")(_forward)
    op.register_fake(_forward_fake)
    back = define(f"{lib}::{name}_backward", mutates_args=(),
                  schema="(Tensor grad, Tensor tokens, SymInt vocab) -> Tensor")(_backward)
    back.register_fake(_backward_fake)

    def _setup(ctx, inputs, output):
        ctx.save_for_backward(inputs[0])
        ctx.vocab = inputs[1].shape[0]

    def _grad(ctx, grad):
        return None, back(grad, ctx.saved_tensors[0], ctx.vocab)

    op.register_autograd(_grad, setup_context=_setup)
    with _lock:
        _OPS[key] = op
    return op
