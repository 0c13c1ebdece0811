"""Online-softmax attention fold: O = softmax(scale * Q K^T [+ causal mask]) V.

There is no reference function for this path (attention-chain fusion is a non-goal of the
reference, docs/roadmap.md:28-30); the fold is the logsumexp skeleton's repair
exp(s - s2) (tests/test_neptune_opt.py:347) applied per key tile to the running
(max, sum, output) state, with MFMA for Q K^T and P V.  The causal mask is torch's
`is_causal=True` (query i sees keys j <= i).  The oracle is the closed form in fp32.

Layout contract: q [B, H, Sq, D], k/v [B, H, Sk, D], D in {64, 128, 256}, one dtype (bf16 or
fp16), unit stride on D; other strides are honoured (rows must be 16-byte aligned, otherwise the
input is made contiguous).  Output is a fresh contiguous [B, H, Sq, D] tensor of the input dtype;
`return_lse` adds the fp32 [B, H, Sq] natural-log logsumexp of the scaled, masked scores.

Calls of at most 16 queries (decoding), and longer ones that `_short_wins` estimates to be cheaper
so (few heads, few keys), run kernels of their own: they split a head's keys over workgroups and
take P and V in fp32 (see SHORT_MAX_SQ).  The MFMA path below is about the others; in both a hidden
key's V reaches no query.

Every input has a result; nothing is refused at run time and no device-side assert is used.
The MFMA path feeds V to the P.V product as fp16 images scaled per 64-key tile by a power of
two (exact for |v| < 2^28 in a tile, see V_EXPONENT_MAX).  A workgroup whose keys include a
tile beyond that (|v| >= 2^28, inf or NaN) recomputes its queries with the kernel's exact fp32
path: O = sum_j p_j v_j / sum_j p_j over the visible keys in IEEE fp32, so only rows that see
a non-finite V value become non-finite.
"""
from __future__ import annotations

import functools
import math
import threading

from neptune_codegen import dispatch, hip
from neptune_codegen.emitters import (ATTN_HEAD_DIMS, ATTN_SHORT_BLOCK_M, ATTN_SHORT_TILE,
                                      ATTN_SHORT_WAVES, BASE_OPTIONS, attention_block_m,
                                      attention_fold_threads, attention_kernel_name,
                                      attention_pack_kernel_name, attention_short_kernel_names,
                                      attention_w64, emit_attention_short_source,
                                      emit_attention_source)

_PROGRAMS: dict = {}
_OPS: dict = {}
_lock = threading.Lock()
LOG2E = 1.4426950408889634
BLOCK_M = 256           # queries per fold workgroup up to head dim 128 (8 waves of 32)
BLOCK_N = 64            # keys per tile (one V^T image per tile)
K_ROW_STRIDE_MAX = 1 << 24   # K rows are addressed with 32-bit byte offsets within a tile
Q_ROW_STRIDE_MAX = 1 << 22   # head dim 128: Q rows, with 32-bit byte offsets within 256 rows
ANY_STRIDE = 1 << 62         # read with 64-bit addresses
# V^T tiles are fp16 images of v * 2^-e, e the tile's exponent (0 below 2^15).  A tile value
# below 2^(e - 14) keeps only an absolute precision of 2^(e - 25), which bounds the error it
# adds to O; e <= 13 keeps that under 2^-12, a quarter of the bf16 absolute tolerance.  Blocks
# of queries that see a larger tile, or inf/NaN in V, take the exact fp32 path.  (fp32
# accumulation of O, |O acc| <= keys * 2^8 * 2^28, cannot overflow at this bound.)
V_EXPONENT_MAX = 13
# Head dim 128 has two fold kernels with bit-identical results: 8 waves x 32 queries
# (compiler-scheduled) and 4 waves x 64 queries (the instruction-scheduled loop of
# attention_asm.py).  The second is faster per key tile (one LDS fragment feeds two MFMAs, the
# softmax issues between them) but has the larger fixed cost per workgroup and idles a SIMD
# whenever one of its waves is past its causal diagonal.  Measured op-time ratios on MI355X
# (graph replays, the two kernels interleaved in one process, two boxes): non-causal 0.93-0.97
# from 512 keys (1.08 at 256); causal 0.957-0.990 from 3072 queries (B*H 32-128), 0.985 at
# 2048 and 1.03 at 1024, 1536 and 2560.
W64_MIN_SK = 512
W64_CAUSAL_MIN_SQ = 3072


def use_w64(head_dim: int, causal: bool, sq: int, sk: int) -> bool:
    """Whether a fold of this shape runs the 64-queries-per-wave kernel."""
    if head_dim != 128:
        return False
    return sq >= W64_CAUSAL_MIN_SQ if causal else sk >= W64_MIN_SK


def _program(head_dim: int, causal: bool, dtype="bfloat16", w64: bool | None = None,
             waves: int | None = None, parts: bool = False) -> hip.Program:
    w64 = attention_w64(head_dim, w64)
    key = (head_dim, causal, str(dtype), w64, waves, parts)
    with _lock:
        prog = _PROGRAMS.get(key)
        if prog is None:
            name = attention_kernel_name(head_dim, causal, dtype, w64, waves, parts)
            prog = hip.Program(emit_attention_source(head_dim, causal, dtype, w64=w64, waves=waves,
                                                     parts=parts), f"{name}.hip", BASE_OPTIONS)
            _PROGRAMS[key] = prog
        return prog


def _short_program(head_dim: int, causal: bool, dtype) -> hip.Program:
    key = ("short", head_dim, causal, str(dtype))
    with _lock:
        prog = _PROGRAMS.get(key)
        if prog is None:
            name = attention_short_kernel_names(head_dim, causal, dtype)[0]
            prog = hip.Program(emit_attention_short_source(head_dim, causal, dtype),
                               f"{name}.hip", BASE_OPTIONS)
            _PROGRAMS[key] = prog
        return prog


# Calls of at most 16 queries run the short-query kernels: K and V are read once, by as many
# workgroups as the keys allow, where the others give a head one workgroup with 240 idle query
# slots and stage V twice.  Measured on MI355X (graph replays, cold; the kernels above -> these):
# bf16 B*H=512 sq=1 sk=3000 d=128 312 -> 128 us (6.1 TB/s of K and V); B*H=32 sq=1 sk=32768 784 ->
# 87; B*H=256 sq=8 sk=4096 201 -> 95; fp16 B*H=64 sq=16 sk=5000 d=64 106 -> 25; B*H=8 sq=4 sk=8192
# d=256 383 -> 23; B*H=8 sq=1 sk=512 20 -> 8.5.
# Longer query ranges take them where `_short_wins` finds them cheaper (few heads, few keys).
SHORT_MAX_SQ = 16
# Chunks of a head's keys: a workgroup's 4 waves pass a 32-key tile in about 0.6 us when each CU
# has one, and a split costs a second launch and its chunks' states (3 us + 0.05 us a chunk).
# `short_chunks` takes the cheapest count; against a sweep of 1 to 64 chunks over fourteen shapes
# it is within 4% of the best but for two (d=64, 4 chunks 25 us for 8 at 20.6; sq=1 sk=8192 B*H=1
# 12.4 for 10.7).  At B*H=32 sk=32768 1 chunk takes 556 us, 8 take 87 and 64 take 94.
# No split makes more than 4096 workgroups (16 per CU, states of at most 68 MB).
SHORT_MAX_CHUNKS, SHORT_MAX_WORKGROUPS = 64, 4096
SHORT_TILE_US, SHORT_MERGE_US, SHORT_CHUNK_US = 0.6, 3.0, 0.05
CUS = 256


def short_chunks(units: int, sk: int) -> tuple[int, int]:
    """(chunks, tiles per chunk) of a head's keys for `units` (head, query block) pairs."""
    return _tile_chunks(units, -(-sk // ATTN_SHORT_TILE))


@functools.lru_cache(maxsize=4096)
def _tile_chunks(units: int, tiles: int) -> tuple[int, int]:
    # kept by tiles: a key range that grows token by token is searched once in 32 calls
    most = max(1, min(SHORT_MAX_CHUNKS, tiles // ATTN_SHORT_WAVES, SHORT_MAX_WORKGROUPS // units))
    best, cost = 1, -(-units // CUS) * tiles * SHORT_TILE_US
    least = max(units * tiles / CUS, -(-tiles // most))     # passes of any split
    for chunks in range(2, most + 1):
        merge = SHORT_MERGE_US + chunks * SHORT_CHUNK_US
        if least * SHORT_TILE_US + merge >= cost:
            break                                # nor is any larger count cheaper
        us = -(-units * chunks // CUS) * -(-tiles // chunks) * SHORT_TILE_US + merge
        if us < cost:
            best, cost = chunks, us
    per = -(-tiles // best)
    return -(-tiles // per), per


# What `_fold_choice` and `_short_wins` price a call with, in us on MI355X, by head dim (fits of
# graph-replayed calls over 24 shapes, cold): one workgroup's pass over a 64-key tile with a CU to
# itself -- the 256-query kernels (two workgroups on a CU pass theirs hardly faster; at head dim 128
# from 1.45 us on a nearly empty chip to 2.05 on a full one, whose clock drops) and the 128-query one
# (4 waves x 32 queries) --, a workgroup's start and readout, and the merge launch with its state's
# traffic.
TILE_256_US = {64: (1.1, 0.0), 128: (1.45, 0.6), 256: None}
TILE_128_US = {64: 0.6, 128: 1.15, 256: 3.3}
BLOCK_US, MERGE_US, STATE_BYTES_PER_US, PACK_US, PACK_BYTES_PER_US = 2.5, 6.0, 8e6, 4.0, 5e6
MAX_STATE_BYTES = 256 << 20
# Heads beyond the 256 MB of the last cache: a head's query blocks are a launch's width apart, so each
# reads its K and V^T from HBM again, the fewer queries in a block, the more often (bf16 full, B*H=640
# sq=601 sk=1184 d=128: 403 us with 256-query blocks, 474 with 128; B*H=1120 s=601 414 and 485; within
# the cache, B*H=640 s=601, 241 and 215).  Causal blocks start with the longest and share more.
CACHE_BYTES, CACHE_BYTES_PER_US = 256 << 20, 5.5e6
# The short-query kernels: launch, a workgroup's start and end, its 4 waves' pass over 4 tiles of
# 32 keys, and the workgroups the chip holds at once.
SHORT_LAUNCH_US, SHORT_BLOCK_US = 3.0, 3.0
SHORT_PASS_US = {64: 1.2, 128: 1.8, 256: 2.5}
SHORT_RESIDENT = {64: 1024, 128: 512, 256: 256}


def _fold_blocks(sq, sk, causal, bm):
    """(query blocks, blocks whose last tile is on the causal diagonal, tiles of the longest block,
    tiles of all blocks) of a head, with query blocks of `bm`."""
    nqb, tiles, step = -(-sq // bm), -(-sk // BLOCK_N), bm // BLOCK_N
    if not causal:
        return nqb, 0, tiles, nqb * tiles
    rising = min(nqb, tiles // step)             # block i sees min(tiles, step * (i + 1))
    return (nqb, rising, min(tiles, step * nqb),
            step * rising * (rising + 1) // 2 + (nqb - rising) * tiles)


def _fold_items(blocks, per, step):
    """Workgroups of a head with its blocks in parts of `per` tiles."""
    nqb, rising, longest, _ = blocks
    items = (nqb - rising) * -(-longest // per)
    for k in range(-(-step * rising // per)):    # rising blocks that have a part k
        items += rising - k * per // step
    return items


def _fold_cost(bh, sq, head_dim, causal, bm, blocks, tile_us, per):
    """us of the fold (and merge) with query blocks of `bm` and keys in parts of `per` tiles."""
    nqb, _, longest, total = blocks
    per = min(per, longest)
    items = bh * _fold_items(blocks, per, bm // BLOCK_N)
    if causal:     # heaviest first: the last items to finish are about half a part apart
        tiles = max(per, bh * total / CUS + per / 2)
    else:
        tiles = -(-items // CUS) * per
    cost = tile_us * tiles + BLOCK_US * max(1.0, items / CUS)
    tile_bytes = bh * BLOCK_N * head_dim * 4           # of K and V^T, over the heads
    if not causal and longest * tile_bytes > CACHE_BYTES:
        cost = max(cost, total * tile_bytes / CACHE_BYTES_PER_US)
    if per < longest:
        state = 2 * 4 * items * sq / nqb * head_dim    # written and read, fp32
        cost += MERGE_US + state / STATE_BYTES_PER_US
    return cost


def _fold_choice(bh: int, sq: int, sk: int, head_dim: int, causal: bool) -> tuple:
    """(us, (w64, waves, tiles per part or None)) of the cheapest fold after the V^T pack.

    The 256-query kernels pass a tile for fewest us per query and are best on a full chip; the
    128-query one makes twice the workgroups, and parts of the keys make as many as it takes.
    Measured, 256 queries / 128 / 128 in parts (us of the whole call): bf16 d=128 full B*H=36
    sq=100 sk=4000 108 / 92 / 44; causal B*H=8 s=4096 103 / 84 / 63; full B*H=64 sq=333 sk=2000
    67 / 57 / 59; causal B*H=128 s=1500 122 / 117 / 162; full B*H=128 s=512 33 / 34 / 64; causal
    B*H=128 s=4096 592 / 645 / -; d=64 causal B*H=1 s=6000 110 / 82 / 28; d=256 full B*H=16 s=700
    - / 45 / 43.

    Found once for the sizes of the same tile counts, so that lengths that change from call to call
    are not searched anew."""
    us, waves, per = _tile_choice(bh, -(-sq // BLOCK_N), -(-sk // BLOCK_N), head_dim, causal)
    return us, (waves == 8 and use_w64(head_dim, causal, sq, sk), waves, per)


@functools.lru_cache(maxsize=4096)
def _tile_choice(bh: int, sq_tiles: int, sk_tiles: int, head_dim: int, causal: bool) -> tuple:
    """(us, waves, tiles per part or None) of the cheapest fold."""
    sq, sk = sq_tiles * BLOCK_N, sk_tiles * BLOCK_N
    most = -(-(min(sk, sq) if causal else sk) // BLOCK_N)
    big = TILE_256_US[head_dim]
    best = None
    if big is not None:
        tile_us = big[0] + big[1] * min(1.0, bh * -(-sq // 256) / CUS)
        best = (_fold_cost(bh, sq, head_dim, causal, 256, _fold_blocks(sq, sk, causal, 256), tile_us,
                           most + 4), 8, None)
    blocks, tile_us = _fold_blocks(sq, sk, causal, 128), TILE_128_US[head_dim]
    # the passes, workgroups and merge of any split
    least = tile_us * (bh * blocks[3] / CUS) + BLOCK_US * max(1.0, bh * blocks[0] / CUS) + MERGE_US
    for parts in (1, 2, 3, 4, 6, 8, 12, 16):
        per = -(-most // parts)
        if parts > 1 and (per < 2 or parts * bh * sq * (head_dim + 2) * 4 > MAX_STATE_BYTES
                          or least >= best[0]):
            break
        cost = _fold_cost(bh, sq, head_dim, causal, 128, blocks, tile_us, per if parts > 1 else most + 4)
        if best is None or cost < best[0]:
            best = (cost, 4, per if parts > 1 else None)
    return best


def _fold_plan(bh, sq, sk, head_dim, causal):
    return _fold_choice(bh, sq, sk, head_dim, causal)[1]


_KERNELS: dict = {}


def _kernels(device, head_dim, causal, dtype, short, w64=None, waves=None, parts=False) -> tuple:
    """(pack or None, fold, merge or None) of one kind of call, fetched once per device."""
    key = (device, head_dim, causal, dtype, short, w64, waves, parts)
    found = _KERNELS.get(key)
    if found is not None:
        return found
    if short:
        names = attention_short_kernel_names(head_dim, causal, dtype)
        prog = _short_program(head_dim, causal, dtype)
        found = (None,
                 prog.kernel(names[0], (hip.PTR,) * 7 + (hip.I32,) * 6 + (hip.I64,) * 9 + (hip.F32,),
                             64 * ATTN_SHORT_WAVES, device),
                 prog.kernel(names[1], (hip.PTR,) * 4 + (hip.I64, hip.I32), 256, device))
    else:
        prog = _program(head_dim, causal, dtype, w64, waves, parts)
        name = attention_kernel_name(head_dim, causal, dtype, w64, waves, parts)
        found = (prog.kernel(attention_pack_kernel_name(head_dim, dtype),
                             (hip.PTR,) * 3 + (hip.I32,) * 2 + (hip.I64,) * 3, 256, device),
                 prog.kernel(name, (hip.PTR,) * 7 + (hip.I32,) * 3 + (hip.I64,) * 9 + (hip.I32, hip.F32)
                             + ((hip.PTR,) * 2 + (hip.I32,) * 2 if parts else ()),
                             attention_fold_threads(head_dim, w64, waves), device),
                 prog.kernel(name + "_merge", (hip.PTR,) * 4 + (hip.I64,) + (hip.I32,) * 3, 256, device)
                 if parts else None)
    _KERNELS[key] = found
    return found


def _short_wins(bh: int, sq: int, sk: int, head_dim: int, causal: bool) -> bool:
    """Whether the short-query kernels run a call: always up to 16 queries; beyond, where they are
    estimated 15% cheaper (bf16 causal B*H=8 s=512 13.3 us against 17.5, d=256 causal B*H=16 s=100
    9.8 against 18.4; B*H=12 s=1000 d=64 full 34 against 21; B*H=160 sq=35 sk=5120 196 against
    189 on 256-query blocks)."""
    return sq <= SHORT_MAX_SQ or _short_cheaper(bh, -(-sq // ATTN_SHORT_BLOCK_M),
                                                -(-sk // ATTN_SHORT_TILE), head_dim, causal)


@functools.lru_cache(maxsize=4096)
def _short_cheaper(bh: int, sq_blocks: int, sk_tiles: int, head_dim: int, causal: bool) -> bool:
    sq, sk = sq_blocks * ATTN_SHORT_BLOCK_M, sk_tiles * ATTN_SHORT_TILE
    seen = min(sq, sk) if causal else sk
    fold = (_fold_choice(bh, sq, sk, head_dim, causal)[0] + PACK_US
            + bh * seen * head_dim * 4 / PACK_BYTES_PER_US)
    units = bh * sq_blocks
    chunks, per = short_chunks(units, seen)
    wait = (SHORT_LAUNCH_US + -(-units * chunks // SHORT_RESIDENT[head_dim])
            * (SHORT_BLOCK_US + -(-per // ATTN_SHORT_WAVES) * SHORT_PASS_US[head_dim]))
    # a full chip passes a 32-key tile per CU in SHORT_TILE_US at head dim 128, whatever is resident
    busy = units * -(-seen // ATTN_SHORT_TILE) / CUS * SHORT_TILE_US * head_dim / 128
    short = max(wait, busy) + (MERGE_US if chunks > 1 else 0.0)
    return 1.15 * short < fold


def validate_attention_inputs(q, k, v, *, metadata: bool = False):
    import torch

    strided, dtypes = torch.strided, (torch.bfloat16, torch.float16)
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        if t.layout != strided:
            raise TypeError(f"attention {nm} must be strided")
        if t.ndim != 4:
            raise ValueError(f"attention {nm} must be [batch, heads, seq, head_dim]")
        if t.dtype not in dtypes:
            raise TypeError(f"attention fold supports bfloat16 and float16 inputs, got {t.dtype} for {nm}")
        if not metadata and t.device.type != "cuda":
            raise ValueError("attention execution requires a ROCm (cuda) device")
    qs, ks = q.shape, k.shape
    if ks != v.shape or qs[0] != ks[0] or qs[1] != ks[1] or qs[3] != ks[3]:
        raise ValueError(f"attention shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"attention q, k, v must share one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.device != k.device or q.device != v.device:
        raise ValueError("attention tensors must be on the same device")
    if qs[3] not in ATTN_HEAD_DIMS:
        raise NotImplementedError("attention fold supports head_dim 64, 128 and 256")
    if ks[2] == 0:
        raise ValueError("attention needs at least one key")
    return tuple(qs)


def _operand(t, row_stride_max):
    """(t, or its contiguous copy where a kernel cannot read its rows; batch, head, row strides)."""
    sb, sh, ss, sd = t.stride()
    if (sd == 1 and sb % 8 == 0 and sh % 8 == 0 and ss % 8 == 0 and ss < row_stride_max
            and t.data_ptr() % 16 == 0):
        return t, (sb, sh, ss)
    t = t.contiguous()
    return t, t.stride()[:3]


def run_attention(q, k, v, *, scale: float | None = None, causal: bool = True,
                  return_lse: bool = False):
    """Attention fold on the current stream; see the module docstring for the contract.

    A call on plain device tensors whose dtypes, devices, shapes, strides, 16-byte alignment and
    options were seen before reuses that call's kernels and launch shapes: everything the
    validation and the launch choice read is in that key, so only the allocations and the launches
    remain (not while launches are recorded)."""
    key = _seen_key(q, k, v, scale, causal, return_lse)
    call = _SEEN.get(key) if key is not None else None
    if call is not None:
        out, lse = call.run(q, k, v)
        return (out, lse) if return_lse else out
    if key is None and _is_metadata(q):    # shapes may be symbolic: no launch is chosen
        out, lse, _, _ = _outputs(q, k, v, scale, return_lse, True)
    elif _takes_short(q, k, causal):
        out, lse, call = _launch_short(q, k, v, scale, causal, return_lse)
    else:
        out, lse, call, _ = _launch_fold(q, k, v, scale, causal, return_lse, V_EXPONENT_MAX)
    if key is not None and call is not None:
        if len(_SEEN) >= _SEEN_MAX:
            _SEEN.clear()
        _SEEN[key] = call
    return (out, lse) if return_lse else out


_SEEN: dict = {}
_SEEN_MAX = 4096


def _seen_key(q, k, v, scale, causal, return_lse):
    """Key of a call on plain strided device tensors, or None where the call takes the full path."""
    import torch

    # a scale whose printed form may not be its value (a tensor) takes the full path
    if hip.recording_active() or not (scale is None or type(scale) in (int, float)):
        return None
    plain, strided = torch.Tensor, torch.strided
    for t in (q, k, v):
        if type(t) is not plain or not t.is_cuda or t.layout != strided:
            return None
    # (a NaN scale equals no key, and is refused)
    return (type(scale), scale, bool(causal), bool(return_lse),
            q.dtype, q.device, q.shape, q.stride(), q.data_ptr() % 16,
            k.dtype, k.device, k.shape, k.stride(), k.data_ptr() % 16,
            v.dtype, v.device, v.shape, v.stride(), v.data_ptr() % 16)


class _Call:
    """The launches of one call layout: kernels, grids and the arguments that are not pointers.
    Pointers, outputs and workspace are each run's own."""

    __slots__ = ("shape", "lse_shape", "nbytes", "exps", "state", "rows_bytes", "pack", "fold", "merge")

    def __init__(self, shape, return_lse):
        self.shape, self.lse_shape = shape, (shape[:3] if return_lse else None)
        self.nbytes = 0                      # workspace: V^T images, exponents, parts' states
        self.exps = self.state = None        # byte offsets of the last two, and of (max, sum)
        self.rows_bytes = 0                  # behind the states' O
        self.pack = self.fold = self.merge = None    # (kernel, grid, further arguments)

    def run(self, q, k, v, out=None, lse=None, exps=None):
        """(out, lse or None); the tile exponents go to `exps` where it is given."""
        import torch

        if out is None:
            out = torch.empty(self.shape, dtype=q.dtype, device=q.device)
            if self.lse_shape is not None:
                lse = torch.empty(self.lse_shape, dtype=torch.float32, device=q.device)
        work = torch.empty(self.nbytes, dtype=torch.uint8, device=q.device) if self.nbytes else None
        base = work.data_ptr() if work is not None else 0
        stream = hip.current_stream(q.device)
        po = pml = 0
        if self.state is not None:
            po = base + self.state
            pml = po + self.rows_bytes
        lse_ptr = lse.data_ptr() if lse is not None else 0
        kernel, grid, rest, tail = self.fold
        if self.pack is None:
            kernel.launch(grid, (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr,
                                 po, pml) + rest, stream)
        else:
            exps_ptr = base + self.exps if exps is None else exps.data_ptr()
            pack, pack_grid, pack_rest = self.pack
            pack.launch(pack_grid, (v.data_ptr(), base, exps_ptr) + pack_rest, stream)
            kernel.launch(grid, (q.data_ptr(), k.data_ptr(), base, exps_ptr, v.data_ptr(), out.data_ptr(),
                                 lse_ptr) + rest + ((po, pml) + tail if tail else ()), stream)
        if self.merge is not None:
            merge, merge_grid, merge_rest = self.merge
            merge.launch(merge_grid, (po, pml, out.data_ptr(), lse_ptr) + merge_rest, stream)
        return out, lse

    def add_state(self, parts, rows, head_dim):
        """Workspace of `parts` fp32 states (O, then (max, sum)) of every query row."""
        self.state = -(-self.nbytes // 256) * 256
        self.rows_bytes = 4 * parts * rows * head_dim
        self.nbytes = self.state + self.rows_bytes + 8 * parts * rows


def _takes_short(q, k, causal) -> bool:
    """Whether the call runs the short-query kernels (calls to be refused do not matter here)."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[3] not in ATTN_HEAD_DIMS or 0 in qs or 0 in ks:
        return False
    return _short_wins(qs[0] * qs[1], qs[2], ks[2], qs[3], bool(causal))


def launch_attention(q, k, v, *, scale: float | None = None, causal: bool = True,
                     return_lse: bool = False):
    """(out, lse or None, exps or None): the V^T pack and the fold.  `exps` is the int32 tile
    exponent table [B*H*ceil(Sk/64)] the pack wrote (None when nothing was launched; of the first
    min(Sk, Sq) keys under the causal mask, which hides the others from every query);
    `exact_path_taken(exps)` tells whether some query block took the exact fp32 path."""
    return _launch(q, k, v, scale, causal, return_lse, V_EXPONENT_MAX)


def _is_metadata(q) -> bool:
    from torch._subclasses.fake_tensor import FakeTensor

    return isinstance(q, FakeTensor) or q.device.type == "meta"


def _outputs(q, k, v, scale, return_lse, metadata):
    """(out, lse or None, scale, whether nothing is to be launched) after validation."""
    import torch

    shape = validate_attention_inputs(q, k, v, metadata=metadata)
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    if metadata or out.numel() == 0:
        return out, lse, scale, True
    scale = 1.0 / math.sqrt(shape[3]) if scale is None else float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("attention scale must be finite and positive")
    return out, lse, scale, False


def _launch_short(q, k, v, scale, causal, return_lse):
    """(out, lse or None, call) through the short-query kernels; the call is None where an input
    was copied."""
    import torch

    out, lse, scale, done = _outputs(q, k, v, scale, return_lse, False)
    if done:
        return out, lse, None
    B, H, Sq, D = q.shape
    given = (q, k, v)
    (q, qs), (k, ks), (v, vs) = (_operand(q, ANY_STRIDE), _operand(k, K_ROW_STRIDE_MAX),
                                 _operand(v, K_ROW_STRIDE_MAX))
    device = q.device.index if q.device.index is not None else torch.cuda.current_device()
    Sk = k.shape[2]
    nqb = -(-Sq // ATTN_SHORT_BLOCK_M)
    chunks, per = short_chunks(B * H * nqb, min(Sk, Sq) if causal else Sk)
    rows = B * H * Sq
    call = _Call(q.shape, return_lse)
    _, fold, merge = _kernels(device, D, bool(causal), q.dtype, True)
    call.fold = (fold, (-(-B * H * chunks // 8) * nqb * 8,),
                 (B, H, Sq, Sk, chunks, per) + qs + ks + vs + (scale * LOG2E,), ())
    if chunks > 1:
        call.add_state(chunks, rows, D)
        call.merge = (merge, (rows,), (rows, chunks))
    call.run(q, k, v, out, lse)
    return out, lse, call if q is given[0] and k is given[1] and v is given[2] else None


def _launch(q, k, v, scale, causal, return_lse, e_max: int, w64: bool | None = None,
            waves: int | None = None, per: int | None = None):
    """(out, lse or None, exps or None) with the exact path's threshold as a parameter: e_max = -1
    sends every query block through the exact fp32 path (the tests compare the two paths with
    it).  The shape picks the fold unless `w64` or `waves` name it: `w64=False` is a
    compiler-scheduled 32-queries-per-wave kernel (8 waves, or `waves`; the keys in parts of
    `per` tiles), whose results at head dim 128 equal the instruction-scheduled one's bit for bit
    when the keys are whole."""
    if _is_metadata(q):
        return _outputs(q, k, v, scale, return_lse, True)[:2] + (None,)
    out, lse, _, exps = _launch_fold(q, k, v, scale, causal, return_lse, e_max, w64, waves, per, True)
    return out, lse, exps


def _launch_fold(q, k, v, scale, causal, return_lse, e_max, w64=None, waves=None, per=None,
                 keep_exps=False):
    """(out, lse or None, call, exponents or None) of the V^T pack and the fold; the call is None
    where an input was copied.  With `keep_exps` the exponents are a tensor of their own: a caller
    that holds on to them holds no workspace."""
    import torch

    out, lse, scale, done = _outputs(q, k, v, scale, return_lse, False)
    if done:
        return out, lse, None, None
    B, H, Sq, D = q.shape
    if w64 is None and waves is None:
        w64, waves, per = _fold_plan(B * H, Sq, k.shape[2], D, bool(causal))
    given = (q, k, v)
    (q, qs), (k, ks), (v, vs) = (_operand(q, Q_ROW_STRIDE_MAX), _operand(k, K_ROW_STRIDE_MAX),
                                 _operand(v, ANY_STRIDE))
    device = q.device.index if q.device.index is not None else torch.cuda.current_device()
    Sk = min(k.shape[2], Sq) if causal else k.shape[2]    # no query sees a key past the last query
    ntiles = (Sk + BLOCK_N - 1) // BLOCK_N
    call = _Call(q.shape, return_lse)
    # V^T tile images (fp16, MFMA operand order) and one power-of-two exponent per tile
    call.exps = B * H * ntiles * D * BLOCK_N * 2
    call.nbytes = call.exps + B * H * ntiles * 4
    w64 = attention_w64(D, w64)
    bm = attention_block_m(D, w64, waves)
    nqb = (Sq + bm - 1) // bm
    parts, rows = 1, B * H * Sq
    if not w64:
        most = -(-(min(Sk, nqb * bm) if causal else Sk) // BLOCK_N)   # tiles of the longest block
        per = min(per or most, most)
        parts = -(-most // per)
    pack, fold, merge = _kernels(device, D, bool(causal), q.dtype, False, w64, waves, parts > 1)
    call.pack = (pack, (B * H * ntiles,), (H, Sk) + vs)
    call.fold = (fold, (nqb * B * H * parts,),
                 (H, Sq, Sk) + qs + ks + vs + (int(e_max), scale * LOG2E),
                 (parts, per) if parts > 1 else ())
    if parts > 1:
        call.add_state(parts, rows, D)
        call.merge = (merge, (-(-rows * (D // 4) // 256),), (rows, Sq, Sk, per))
    exps = torch.empty(B * H * ntiles, dtype=torch.int32, device=q.device) if keep_exps else None
    call.run(q, k, v, out, lse, exps)
    copied = q is not given[0] or k is not given[1] or v is not given[2]
    return out, lse, None if copied else call, exps


def exact_path_taken(exps) -> bool:
    """Host check (synchronises): some V tile was beyond the MFMA path's range, so the query
    blocks that see it were computed by the exact fp32 path."""
    return bool((exps > V_EXPONENT_MAX).any().item())


attention_fold = run_attention


@dispatch.one_at_a_time
def as_attention_op(scale: float | None = None, causal: bool = True, lib: str = "neptune"):
    """Custom op `(Tensor q, Tensor k, Tensor v) -> Tensor` with scale and mask in its name."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    params = {"scale": float(scale)} if scale is not None else {}
    key = (lib, tuple(sorted(params.items())), causal)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"attention_fold{parameter_tag(params)}_{'causal' if causal else 'full'}"

    def _impl(q, k, v):
        return run_attention(q, k, v, scale=scale, causal=causal)

    def _fake(q, k, v):
        validate_attention_inputs(q, k, v, metadata=True)
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)

    op = torch.library.custom_op(f"{lib}::{name}", mutates_args=(),
                                 schema="(Tensor q, Tensor k, Tensor v) -> Tensor")(_impl)
    op.register_fake(_fake)
    with _lock:
        _OPS[key] = op
    return op
