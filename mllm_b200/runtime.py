"""Python mirror of mLLM's stateless runtime API for the attention path, on the B200 kernels.

Same names, argument meaning and error behaviour as the reference's C++ classes
(src/core/runtime/{KVCache,RoPE,Attention,TransformerBlock}.h); every device computation goes
through the C ABI of libmllm_attn.so (include/mllm_attn.h).  Projections (Linear) stay torch
GEMMs, exactly as the reference keeps them in LibTorch.  There is no CPU path: CUDA bf16
tensors are required and anything else raises RuntimeError, like the reference's checks.

  KVCache                 src/core/runtime/KVCache.h:9-28  -- preallocated bf16 rows instead of
                          a tensor grown by torch::cat; .key/.value are views of the valid rows
  RoPE.build_cos_sin      src/core/runtime/RoPE.h:29-59
  RoPE.apply              src/core/runtime/RoPE.h:68-89
  Attention.forward       src/core/runtime/Attention.h:29-86
  Attention.forward_projected  src/core/runtime/Attention.h:100-326 (+ optional fused QK-norm,
                          which the reference does in TransformerBlock.h:103-134)
  PagedKVCache8           8-bit paged cache (no reference counterpart): the functions below take it
                          wherever they take a PagedKVCache
  attention_block         the attention half of TransformerBlock::Forward (h -> attention out)
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import abi

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn


def _check_cuda_bf16(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: the B200 attention path needs CUDA tensors (no CPU fallback)")
    if t.dtype != BF16:
        raise RuntimeError(f"{name}: expected bfloat16, got {t.dtype}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


class KVCache:
    """Per-layer KV cache: bf16 rows [batch, num_kv_heads, capacity, head_dim] written in place.

    Mirrors KVCache.h:9-28: `key`/`value` are the valid rows [B, Hkv, L, D] (views), so callers
    that read `key.size(2)` (the runners' decode position, QwenRunner.cpp:301-310) see the
    cache length.  `lengths` holds per-sequence lengths for ragged batches."""

    capture_max_len = None   # set while a CUDA graph of decode steps is captured (decode_step)

    def __init__(self, batch: int, num_kv_heads: int, head_dim: int, capacity: int,
                 device="cuda", zero: bool = True):
        alloc = torch.zeros if zero else torch.empty
        self.key_buf = alloc((batch, num_kv_heads, capacity, head_dim), dtype=BF16, device=device)
        self.value_buf = alloc((batch, num_kv_heads, capacity, head_dim), dtype=BF16, device=device)
        self.capacity = capacity
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._host_lengths = [0] * batch

    # -- reference API --
    def is_initialized(self) -> bool:
        return max(self._host_lengths) > 0

    def clear(self) -> None:
        self.lengths.zero_()
        self._host_lengths = [0] * len(self._host_lengths)

    @property
    def length(self) -> int:
        if len(set(self._host_lengths)) != 1:
            raise RuntimeError("KVCache: ragged batch has no single length")
        return self._host_lengths[0]

    @property
    def key(self) -> torch.Tensor:
        return self.key_buf[:, :, : self.length]

    @property
    def value(self) -> torch.Tensor:
        return self.value_buf[:, :, : self.length]

    # -- layout for the kernels --
    @property
    def strides(self):
        s = self.key_buf.stride()
        return s[0], s[1], s[2]

    def host_lengths(self) -> list[int]:
        return list(self._host_lengths)

    def advance(self, n: int | list[int]) -> None:
        add = n if isinstance(n, list) else [n] * len(self._host_lengths)
        self._host_lengths = [a + b for a, b in zip(self._host_lengths, add)]
        if max(self._host_lengths) > self.capacity:
            raise RuntimeError("KVCache: capacity exceeded")
        self.lengths.copy_(torch.tensor(self._host_lengths, dtype=torch.int32), non_blocking=True)

    def set_lengths(self, lens: list[int]) -> None:
        if max(lens) > self.capacity:
            raise RuntimeError("KVCache: capacity exceeded")
        self._host_lengths = list(lens)
        self.lengths.copy_(torch.tensor(lens, dtype=torch.int32), non_blocking=True)

    def advance_host(self, n: int, batch: int) -> None:
        """The host copy of the lengths after a replayed decode graph advanced the device copy."""
        for b in range(batch):
            self._host_lengths[b] += n


class RoPE:
    @staticmethod
    def build_cos_sin(positions: torch.Tensor, head_dim: int, rope_theta: float):
        """RoPE::BuildCosSin: (cos, sin) fp32 [S, D] on the positions' device."""
        if head_dim % 2 != 0:
            raise RuntimeError("RoPE: head_dim must be even.")
        if not positions.is_cuda:
            raise RuntimeError("RoPE: positions must be a CUDA tensor (no CPU fallback)")
        pos = positions.to(torch.int64).contiguous()
        n = pos.numel()
        cos = torch.empty((n, head_dim), dtype=torch.float32, device=pos.device)
        sin = torch.empty_like(cos)
        abi.call("mllm_rope_build_cos_sin", _ptr(pos), n, head_dim, float(rope_theta), _ptr(cos),
                 _ptr(sin), abi.stream_handle())
        return cos, sin

    @staticmethod
    def apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """RoPE::Apply for bf16 x [B, H, S, D] (any strides with D contiguous)."""
        _check_cuda_bf16("RoPE", x)
        if x.dim() != 4 or x.stride(3) != 1:
            raise RuntimeError("RoPE: x must be [B, H, S, D] with D contiguous")
        B, H, S, D = x.shape
        cos = cos.to(torch.float32).contiguous()
        sin = sin.to(torch.float32).contiguous()
        out = torch.empty((B, H, S, D), dtype=BF16, device=x.device)
        abi.call("mllm_rope_apply_bf16", _ptr(x), x.stride(0), x.stride(1), x.stride(2), B, H, S, D,
                 _ptr(cos), _ptr(sin), _ptr(out), abi.stream_handle())
        return out


class PagedKVCache:
    """Paged KV cache for one layer (the mllm_paged_kv layout): K and V pools of `num_blocks`
    blocks, each `block_size` rows for every kv head ([num_blocks, Hkv, block_size, D] bf16), and
    per-sequence block tables and lengths.  Sequences of any length share the pool without
    padding to the longest.  Blocks are handed out from a free list as sequences grow (`reserve`)
    and zeroed when freed (`release`), so the rows past a sequence's length in its last block are
    always finite.  The reference's KVCache (KVCache.h:9-28) is one contiguous tensor per layer;
    this is the serving-format step beyond it."""

    capture_max_len = None   # set while a CUDA graph of decode steps is captured (decode_step)
    shared_prefix = 0        # rows that the sequences of a decode step were forked with (decode_step)

    def __init__(self, num_blocks: int, num_kv_heads: int, head_dim: int, block_size: int = 256,
                 max_seqs: int = 64, max_blocks_per_seq: int | None = None, device="cuda"):
        if block_size <= 0 or block_size % 128 != 0:
            raise RuntimeError("PagedKVCache: block_size must be a positive multiple of 128")
        self.block_size = block_size
        self.num_blocks = num_blocks
        self.max_blocks_per_seq = max_blocks_per_seq or num_blocks
        self.k_pool = torch.zeros((num_blocks, num_kv_heads, block_size, head_dim), dtype=BF16, device=device)
        self.v_pool = torch.zeros_like(self.k_pool)
        self.block_table = torch.zeros((max_seqs, self.max_blocks_per_seq), dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self._blocks = [[] for _ in range(max_seqs)]
        self._host_lengths = [0] * max_seqs
        self._free = list(range(num_blocks - 1, -1, -1))   # pop() hands out block 0 first
        self._owners = [0] * num_blocks                     # sequences whose table holds the block (fork)
        # per sequence (line, rows): its first `rows` rows are those of that line, the last one being its own.  Sequences
        # that hold a line in common have the rows in common up to the smaller number.
        self._lines = [[(b, math.inf)] for b in range(max_seqs)]
        self._next_line = max_seqs

    @property
    def capacity(self) -> int:
        """Rows one sequence can hold."""
        return self.max_blocks_per_seq * self.block_size

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    def blocks_of(self, seq: int) -> list[int]:
        return list(self._blocks[seq])

    def reserve(self, seq: int, rows: int) -> None:
        """Make sure sequence `seq` has blocks for `rows` rows."""
        need = -(-rows // self.block_size)
        if need > self.max_blocks_per_seq:
            raise RuntimeError("PagedKVCache: sequence exceeds max_blocks_per_seq * block_size rows")
        blocks = self._blocks[seq]
        if need > len(blocks):
            if need - len(blocks) > len(self._free):
                raise RuntimeError("PagedKVCache: out of blocks")
            start = len(blocks)
            while len(blocks) < need:
                blocks.append(self._take_block())
            if need - start == 1:   # a growing sequence's next block: a fill, with no copy from the host to wait for
                self.block_table[seq, start] = blocks[start]
            else:
                self.block_table[seq, start:need] = torch.tensor(blocks[start:need], dtype=torch.int32)

    def _take_block(self) -> int:
        blk = self._free.pop()
        self._owners[blk] = 1
        return blk

    def fork(self, src: int, dst: int, rows: int) -> None:
        """Give the empty row `dst` the first `rows` rows of sequence `src`: it shares src's full blocks
        (a block is freed when its last owner is) and gets a copy of the rows in a block that ends
        inside, as they are now: rows that are reserved and written later reach it in full blocks only.
        Shared rows must not be written again; appending to either sequence does not, and neither
        can be shortened into a block they share (release it instead)."""
        if src == dst or self._blocks[dst] or self._host_lengths[dst]:
            raise RuntimeError("PagedKVCache: fork target row is not empty")
        full, part = divmod(rows, self.block_size)
        if rows < 0 or len(self._blocks[src]) < full + (part > 0):
            raise RuntimeError("PagedKVCache: fork of rows the source does not hold")
        if part and not self._free:
            raise RuntimeError("PagedKVCache: out of blocks")
        blocks = self._blocks[src][:full]
        for blk in blocks:
            self._owners[blk] += 1
        if part:
            blocks.append(self._take_block())
            self._copy_rows(self._blocks[src][full], blocks[-1], part)
        self._blocks[dst] = blocks
        same = rows if self._host_lengths[src] >= rows else full * self.block_size
        self._lines[dst] = [(i, min(n, same)) for i, n in self._lines[src] if same > 0] + self._own_line()
        self.block_table[dst, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
        self._host_lengths[dst] = rows
        self.lengths[dst] = rows

    def _own_line(self) -> list:
        self._next_line += 1
        return [(self._next_line - 1, math.inf)]

    def _rows_in_common(self, batch: int, rows: int, first: int = 0) -> bool:
        """Whether sequences first .. first + batch - 1 came by their first `rows` rows together (fork)."""
        lines = self._lines[first:first + batch]
        return any(n >= rows and all((i, n) in line or any(j == i and m >= rows for j, m in line) for line in lines)
                   for i, n in lines[0])

    def _copy_rows(self, src: int, dst: int, rows: int) -> None:
        for pool in (self.k_pool, self.v_pool):
            pool[dst, :, :rows] = pool[src, :, :rows]

    def release(self, seq: int) -> None:
        """Return sequence `seq`'s blocks to the pool (zeroed), those that no other sequence shares, and
        reset its length."""
        blocks = []
        for blk in self._blocks[seq]:
            self._owners[blk] -= 1
            if self._owners[blk] == 0:
                blocks.append(blk)
        if blocks:
            idx = torch.tensor(blocks, dtype=torch.long, device=self.k_pool.device)
            self._zero_blocks(idx)
            self._free.extend(reversed(blocks))
        self._blocks[seq] = []
        self._lines[seq] = self._own_line()
        self._host_lengths[seq] = 0
        self.lengths[seq] = 0

    def _zero_blocks(self, idx: torch.Tensor) -> None:
        self.k_pool.index_fill_(0, idx, 0)
        self.v_pool.index_fill_(0, idx, 0)

    def move(self, src: int, dst: int) -> None:
        """Hand sequence `src`'s blocks and length to the empty row `dst` (its block-table row is
        copied; no K/V row moves).  A serving loop uses it to keep its live sequences in rows
        0..n-1 when one in the middle finishes."""
        if src == dst:
            return
        if self._blocks[dst] or self._host_lengths[dst]:
            raise RuntimeError("PagedKVCache: move target row is not empty")
        self.block_table[dst].copy_(self.block_table[src])
        self.lengths[dst] = self.lengths[src]
        self._blocks[dst], self._blocks[src] = self._blocks[src], []
        self._lines[dst], self._lines[src] = self._lines[src], self._own_line()
        self._host_lengths[dst], self._host_lengths[src] = self._host_lengths[src], 0
        self.lengths[src] = 0

    def slot(self, seq: int, count: int = 1) -> "PagedSlot":
        """A view of rows seq .. seq + count - 1 as a batch of `count` (prefill of new requests
        while other rows are live)."""
        return PagedSlot(self, seq, count)

    def _shorten(self, lens: list[int], first: int = 0) -> None:
        """For sequences from `first` on that `lens` takes back: refuses a length that falls into a block others share, since
        the next append would write their rows; what lies behind will be written anew, so that the rows in common with
        others end there."""
        short = [(b, n) for b, n in enumerate(lens, first) if n < self._host_lengths[b]]
        for b, n in short:
            at, blocks = n // self.block_size, self._blocks[b]
            if at < len(blocks) and self._owners[blocks[at]] > 1:
                raise RuntimeError("PagedKVCache: a sequence cannot be shortened into a block that others share")
        for b, n in short:
            line = self._lines[b][-1][0]
            old = [(i, min(m, n)) for i, m in self._lines[b] if n > 0]
            known = any(i == line for c, other in enumerate(self._lines) if c != b for i, _ in other)
            self._lines[b] = old + self._own_line() if known else old[:-1] + [(line, math.inf)]

    # -- the KVCache interface the attention functions use --
    def host_lengths(self) -> list[int]:
        return list(self._host_lengths)

    def set_lengths(self, lens: list[int]) -> None:
        self._shorten(lens)
        for b, n in enumerate(lens):
            self.reserve(b, n)
        self._host_lengths[:len(lens)] = list(lens)
        self.lengths[:len(lens)].copy_(torch.tensor(lens, dtype=torch.int32), non_blocking=True)

    def advance(self, n: int | list[int], batch: int | None = None) -> None:
        B = batch if batch is not None else (len(n) if isinstance(n, list) else len(self._host_lengths))
        add = n if isinstance(n, list) else [n] * B
        self.set_lengths([self._host_lengths[b] + add[b] for b in range(B)])

    def advance_host(self, n: int, batch: int) -> None:
        """The host copy of the lengths after a replayed decode graph advanced the device copy
        (the blocks were reserved before the graph was captured)."""
        for b in range(batch):
            self._host_lengths[b] += n

    def length_of(self, batch: int) -> int:
        lens = set(self.host_lengths()[:batch])
        if len(lens) != 1:
            raise RuntimeError("PagedKVCache: ragged batch has no single length")
        return lens.pop()

    def descriptor(self) -> abi.PagedKV:
        s = self.k_pool.stride()
        return abi.PagedKV(self.k_pool.data_ptr(), self.v_pool.data_ptr(), s[0], s[1], s[2], self.num_blocks,
                           self.block_size, self.block_table.data_ptr(), self.block_table.stride(0),
                           self.max_blocks_per_seq)

    def gather(self, seq: int, rows: int):
        """K and V rows [Hkv, rows, D] of sequence `seq`, copied out of the pool (for tests)."""
        blocks = self._blocks[seq][: -(-rows // self.block_size)]
        k = torch.cat([self.k_pool[b] for b in blocks], dim=1)[:, :rows]
        v = torch.cat([self.v_pool[b] for b in blocks], dim=1)[:, :rows]
        return k, v


class PagedSlot(PagedKVCache):
    """Rows `seq` .. `seq + count - 1` of a PagedKVCache seen as a batch of `count`: the same
    pools, the parent's block-table rows and lengths (shared memory), and reserve/advance acting
    on those rows."""

    def __init__(self, parent: PagedKVCache, seq: int, count: int = 1):   # no pool allocation: a view
        if count < 1 or seq < 0 or seq + count > parent.block_table.shape[0]:
            raise RuntimeError("PagedSlot: rows outside the parent cache")
        self._parent, self._seq, self._count = parent, seq, count
        self.block_size = parent.block_size
        self.num_blocks = parent.num_blocks
        self.max_blocks_per_seq = parent.max_blocks_per_seq
        self.k_pool, self.v_pool = parent.k_pool, parent.v_pool
        self.block_table = parent.block_table[seq:seq + count]
        self.lengths = parent.lengths[seq:seq + count]

    def _row(self, seq: int) -> int:
        if not 0 <= seq < self._count:
            raise RuntimeError("PagedSlot: sequence outside the view")
        return self._seq + seq

    @property
    def free_blocks(self) -> int:
        return self._parent.free_blocks

    def blocks_of(self, seq: int) -> list[int]:
        return self._parent.blocks_of(self._row(seq))

    def reserve(self, seq: int, rows: int) -> None:
        self._parent.reserve(self._row(seq), rows)

    def release(self, seq: int = 0) -> None:
        self._parent.release(self._row(seq))

    def fork(self, src: int, dst: int, rows: int) -> None:
        self._parent.fork(self._row(src), self._row(dst), rows)

    def move(self, src: int, dst: int) -> None:
        raise RuntimeError("PagedSlot: move rows on the parent cache")

    def _rows_in_common(self, batch: int, rows: int, first: int = 0) -> bool:
        return self._parent._rows_in_common(batch, rows, self._seq + first)

    def host_lengths(self) -> list[int]:
        return self._parent.host_lengths()[self._seq:self._seq + self._count]

    def set_lengths(self, lens: list[int]) -> None:
        if len(lens) > self._count:
            raise RuntimeError("PagedSlot: more lengths than sequences in the view")
        self._parent._shorten(lens, self._seq)
        for b, n in enumerate(lens):
            self._parent.reserve(self._seq + b, n)
            self._parent._host_lengths[self._seq + b] = n
        self.lengths[:len(lens)].copy_(torch.tensor(lens, dtype=torch.int32), non_blocking=True)

    def advance(self, n, batch: int | None = None) -> None:
        B = batch if batch is not None else (len(n) if isinstance(n, list) else self._count)
        add = n if isinstance(n, list) else [n] * B
        cur = self.host_lengths()
        self.set_lengths([cur[b] + add[b] for b in range(B)])

    def gather(self, seq: int, rows: int):
        return self._parent.gather(self._row(seq), rows)


class PagedKVCache8(PagedKVCache):
    """PagedKVCache whose rows are held in 8 bits (the mllm_paged_kv8 layout): e4m3 values
    [num_blocks, Hkv, block_size, D] and one exponent byte per row [num_blocks, Hkv, block_size],
    a little over half the memory and the decode time of the bf16 cache.  A row stands for
    value * 2^(exponent - 127); rows are quantised as they are appended."""

    def __init__(self, num_blocks: int, num_kv_heads: int, head_dim: int, block_size: int = 256,
                 max_seqs: int = 64, max_blocks_per_seq: int | None = None, device="cuda"):
        # the base class with pools of no size: its block bookkeeping is the same
        super().__init__(num_blocks, num_kv_heads, 0, block_size, max_seqs, max_blocks_per_seq, device)
        shape = (num_blocks, num_kv_heads, block_size)
        self.k_pool = torch.zeros((*shape, head_dim), dtype=torch.uint8, device=device).view(FP8)
        self.v_pool = torch.zeros((*shape, head_dim), dtype=torch.uint8, device=device).view(FP8)
        self.k_exp = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.v_exp = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.one_each = torch.arange(max_seqs + 1, dtype=torch.int32, device=device)   # cu_seqlens of a decode step

    def _zero_blocks(self, idx: torch.Tensor) -> None:
        for t in (self.k_pool.view(torch.uint8), self.v_pool.view(torch.uint8), self.k_exp, self.v_exp):
            t.index_fill_(0, idx, 0)

    def _copy_rows(self, src: int, dst: int, rows: int) -> None:
        for t in (self.k_pool.view(torch.uint8), self.v_pool.view(torch.uint8), self.k_exp, self.v_exp):
            t[dst, :, :rows] = t[src, :, :rows]

    def slot(self, seq: int, count: int = 1) -> "PagedSlot8":
        return PagedSlot8(self, seq, count)

    def descriptor(self) -> abi.PagedKV8:
        s, e = self.k_pool.stride(), self.k_exp.stride()
        if self.v_pool.stride() != s or self.v_exp.stride() != e:
            raise RuntimeError("PagedKVCache8: K and V pools must have the same layout")
        return abi.PagedKV8(self.k_pool.data_ptr(), self.v_pool.data_ptr(), s[0], s[1], s[2], self.k_exp.data_ptr(),
                            self.v_exp.data_ptr(), e[0], e[1], self.num_blocks, self.block_size,
                            self.block_table.data_ptr(), self.block_table.stride(0), self.max_blocks_per_seq)

    def gather(self, seq: int, rows: int):
        """K and V rows [Hkv, rows, D] of sequence `seq` as fp32 values (for tests)."""
        idx = torch.tensor(self.blocks_of(seq)[: -(-rows // self.block_size)], dtype=torch.long,
                           device=self.k_pool.device)
        out = []
        for pool, exps in ((self.k_pool, self.k_exp), (self.v_pool, self.v_exp)):
            v = pool.view(torch.uint8)[idx].view(FP8).float().transpose(0, 1).flatten(1, 2)[:, :rows]
            e = exps[idx].transpose(0, 1).flatten(1, 2)[:, :rows]
            out.append(torch.ldexp(v, (e.int() - 127).unsqueeze(-1)))
        return out[0], out[1]


class PagedSlot8(PagedSlot, PagedKVCache8):
    """PagedSlot of an 8-bit cache."""

    def __init__(self, parent: PagedKVCache8, seq: int, count: int = 1):
        PagedSlot.__init__(self, parent, seq, count)
        self.k_exp, self.v_exp, self.one_each = parent.k_exp, parent.v_exp, parent.one_each

    def gather(self, seq: int, rows: int):
        return PagedKVCache8.gather(self, seq, rows)


class DecodeWorkspace:
    """Grow-only, zero-filled device scratch for the split-K decode partials (the C ABI never
    allocates).  Its 256-byte header must start at zero; every call leaves it zero."""

    def __init__(self):
        self.buf = None

    def get(self, nbytes: int, device) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < nbytes or self.buf.device != torch.device(device):
            self.buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
        return self.buf


_WS = DecodeWorkspace()


class GraphScratch:
    """Device scratch owned by one captured CUDA graph: the decode and projection workspaces
    its kernels were recorded with.  The module's shared workspaces grow by reallocation, which
    would leave a graph writing into freed memory; these buffers live as long as the graph
    (hold the object beside it) and are never replaced while a capture is recording."""

    def __init__(self):
        self._keep: list[torch.Tensor] = []
        self._cur: dict = {}

    def get(self, key: str, nbytes: int, device) -> torch.Tensor:
        buf = self._cur.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            self._keep.append(buf)      # an earlier, smaller one stays alive for the nodes that use it
            self._cur[key] = buf
        return buf


_capture_scratch: GraphScratch | None = None


class graph_scratch:
    """`with graph_scratch(s):` around a CUDA graph capture makes the kernels recorded inside it
    take their workspaces from `s`."""

    def __init__(self, scratch: GraphScratch):
        self.scratch = scratch

    def __enter__(self):
        global _capture_scratch
        self.prev, _capture_scratch = _capture_scratch, self.scratch
        return self.scratch

    def __exit__(self, *exc):
        global _capture_scratch
        _capture_scratch = self.prev
        return False


def _capturing() -> bool:
    if not torch.cuda.is_available() or not torch.cuda.is_current_stream_capturing():
        return False
    if _capture_scratch is None:
        raise RuntimeError("capturing a CUDA graph of these kernels needs runtime.graph_scratch")
    return True


def _check_vec(name: str, t: torch.Tensor, n: int, dtype, dev: int) -> None:
    """A contiguous vector of exactly n elements on CUDA device number `dev`."""
    if t.get_device() != dev or t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise RuntimeError(f"{name}: expected a contiguous {dtype} tensor of {n} elements on cuda:{dev}")


def _launch(dev: int, name: str, *args) -> None:
    """abi.call with torch's current stream of device number `dev` as the last argument; the library launches on
    the current device, so `dev` is made that around the call if it is not."""
    if dev == torch._C._cuda_getDevice():   # the callers hold CUDA tensors: CUDA is initialised
        abi.call(name, *args, torch._C._cuda_getCurrentRawStream(dev) or None)
    else:
        with torch.cuda.device(dev):
            abi.call(name, *args, abi.stream_handle())


@functools.lru_cache(maxsize=256)
def _workspace_size(name: str, *sizes: int) -> int:
    """Bytes a *_workspace_size entry point asks for (it depends on its arguments alone)."""
    return getattr(abi.load(), name)(*sizes)


def qkv_epilogue_kv8(q, k, v, kv_cache: PagedKVCache8, cu_seqlens: torch.Tensor, start: torch.Tensor, positions=None,
                     rope_theta: float = 1e4, rope_table=None, q_norm_weight=None, k_norm_weight=None,
                     eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """The QKV epilogue over an 8-bit cache: per-head QK-RMSNorm (optional), RoPE, and the
    quantising append of K and V.  q [T, H, D], k/v [T, Hkv, D] bf16 (strided views of the
    projections, D contiguous); sequence b owns the tokens cu_seqlens[b] .. cu_seqlens[b+1] - 1
    (int32 device [n + 1]) and they go to its cache rows from start[b] (int32 device [n]) on, whose
    blocks must be reserved; tokens behind the last sequence are left out.  Angles: rope_table =
    (cos, sin) fp32 [T, D], or positions int64 [T] and rope_theta.  Returns Q [T, H, D] (rotated);
    `out` takes it in another layout.  The cache's lengths are the caller's to advance; the
    functions below do both."""
    _check_cuda_bf16("q", q)
    _check_cuda_bf16("k", k)
    _check_cuda_bf16("v", v)
    if not isinstance(kv_cache, PagedKVCache8):
        raise RuntimeError("qkv_epilogue_kv8: needs a PagedKVCache8")
    shape, kv_shape, pool = q.shape, k.shape, kv_cache.k_pool
    q_stride, k_stride, v_stride = q.stride(), k.stride(), v.stride()
    if len(shape) != 3 or len(kv_shape) != 3 or v.shape != kv_shape or \
            q_stride[2] != 1 or k_stride[2] != 1 or v_stride[2] != 1:
        raise RuntimeError("Attention: q, k and v must be rank-3 [T, h, D] with D contiguous")
    T, H, D = shape
    dev = q.get_device()
    Hkv = kv_shape[1]
    if kv_shape[0] != T or kv_shape[2] != D:
        raise RuntimeError("Attention: k and v must be [T, num_kv_heads, D] for q's T and D")
    pool_shape = pool.shape
    if pool_shape[1] != Hkv or pool_shape[3] != D:
        raise RuntimeError("Attention: the cache has other kv heads or another head_dim")
    if k.get_device() != dev or v.get_device() != dev or pool.get_device() != dev:
        raise RuntimeError("Attention: q, k, v and the cache must be on one device")
    n = start.numel()
    if n > kv_cache.block_table.shape[0]:
        raise RuntimeError("Attention: more sequences than the cache has rows for")
    _check_vec("cu_seqlens", cu_seqlens, n + 1, torch.int32, dev)
    _check_vec("start", start, n, torch.int32, dev)
    pos = cos = sin = None
    if rope_table is not None:
        cos, sin = rope_table
        for t in (cos, sin):
            if t.get_device() != dev or t.dtype is not torch.float32 or t.shape != (T, D) or not t.is_contiguous():
                raise RuntimeError("RoPE: tables must be contiguous fp32 [T, D] on q's device")
        cos, sin = cos.data_ptr(), sin.data_ptr()
    else:
        if positions is None:
            raise RuntimeError("RoPE: positions or rope_table required")
        _check_vec("positions", positions, T, torch.int64, dev)
        pos = positions.data_ptr()
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise RuntimeError("Attention: give both q/k norm weights or neither")
    qn = kn = None
    if q_norm_weight is not None:
        qn, kn = q_norm_weight, k_norm_weight
        if qn.dtype is not BF16 or kn.dtype is not BF16 or not qn.is_contiguous() or not kn.is_contiguous():
            qn, kn = qn.to(BF16).contiguous(), kn.to(BF16).contiguous()
        _check_vec("q_norm_weight", qn, D, BF16, dev)
        _check_vec("k_norm_weight", kn, D, BF16, dev)
    if out is None:
        out = torch.empty_strided(shape, (H * D, D, 1), dtype=BF16, device=q.device)   # torch.empty takes 1 us longer
    elif out.shape != shape or out.dtype is not BF16 or out.get_device() != dev or out.stride(2) != 1:
        raise RuntimeError("Attention: out must be bf16 [T, H, D] with D contiguous on q's device")
    out_stride = out.stride()
    _launch(dev, "mllm_qkv_epilogue_varlen_paged_kv8", q.data_ptr(), q_stride[0], q_stride[1], k.data_ptr(), k_stride[0],
            k_stride[1], v.data_ptr(), v_stride[0], v_stride[1], T, H, Hkv, D, pos, rope_theta, cos, sin, _ptr(qn), _ptr(kn),
            eps, out.data_ptr(), out_stride[0], out_stride[1], C.byref(kv_cache.descriptor()), cu_seqlens.data_ptr(), n, start.data_ptr())
    return out


def kv8_read(kv_cache: PagedKVCache8, lens: torch.Tensor, rows: int, first: torch.Tensor | None = None):
    """Cached rows as bf16, exactly: rows first[b] (default 0) .. lens[b] - 1 of sequence b (int32
    device vectors) at rows 0 .. of its part of K and V [n, Hkv, rows, D]; rows past the end of a
    sequence are zero."""
    if not isinstance(kv_cache, PagedKVCache8):
        raise RuntimeError("kv8_read: needs a PagedKVCache8")
    pool = kv_cache.k_pool
    dev = pool.get_device()
    n = lens.numel()
    if rows < 0 or n > kv_cache.block_table.size(0):
        raise RuntimeError("kv8_read: negative rows, or more sequences than the cache has rows for")
    _check_vec("lens", lens, n, torch.int32, dev)
    if first is not None:
        _check_vec("first", first, n, torch.int32, dev)
    Hkv, D = pool.size(1), pool.size(3)
    k = torch.empty_strided((n, Hkv, rows, D), (Hkv * rows * D, rows * D, D, 1), dtype=BF16, device=pool.device)
    v = torch.empty_like(k)
    _launch(dev, "mllm_kv8_read_bf16", C.byref(kv_cache.descriptor()), _ptr(first), lens.data_ptr(), n, Hkv, D, rows,
            k.data_ptr(), v.data_ptr(), Hkv * rows * D, rows * D, D)
    return k, v


def _decode_args(q: torch.Tensor, kv_cache: PagedKVCache, num_kv_heads: int, max_kv_len: int | None):
    """Decode queries [B, H, D] or [B, H, 1, D] checked against a paged cache: (q as 16-byte aligned contiguous
    [B, H, D], its shape, device number, bound on the lengths)."""
    _check_cuda_bf16("q", q)
    shape = q.shape
    if len(shape) == 4 and shape[2] == 1:
        q = q.squeeze(2)
        shape = q.shape
    if len(shape) != 3:
        raise RuntimeError("Attention: decode queries must be [B, H, D] or [B, H, 1, D]")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    pool = kv_cache.k_pool
    dev = pool.get_device()
    pool_shape = pool.shape
    if q.get_device() != dev:
        raise RuntimeError("Attention: q and the cache must be on one device")
    if pool_shape[1] != num_kv_heads or pool_shape[3] != shape[2] or shape[0] > kv_cache.block_table.shape[0]:
        raise RuntimeError("Attention: the cache has other kv heads, another head_dim or fewer sequences")
    L = max_kv_len or max(kv_cache.host_lengths()[:shape[0]], default=0)
    return q, shape, dev, max(min(L, kv_cache.capacity), 1)


def _decode_kv8(q: torch.Tensor, kv_cache: PagedKVCache8, num_kv_heads: int, max_kv_len: int | None) -> torch.Tensor:
    """decode_attention over an 8-bit cache."""
    q, (B, H, D), dev, L = _decode_args(q, kv_cache, num_kv_heads, max_kv_len)
    device = q.device
    out = torch.empty_strided((B, 1, H * D), (H * D, H * D, 1), dtype=BF16, device=device)
    # a workspace of the call's own, from torch's stream-ordered allocator (a captured graph's from its pool)
    nbytes = _workspace_size("mllm_decode_attention_kv8_workspace_size", B, H, num_kv_heads, D)
    ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=device)
    _launch(dev, "mllm_decode_attention_paged_kv8", q.data_ptr(), C.byref(kv_cache.descriptor()), kv_cache.lengths.data_ptr(),
            B, H, num_kv_heads, D, L, 1.0 / math.sqrt(D), out.data_ptr(), ws.data_ptr(), nbytes)
    return out


def _flat_tokens(t: torch.Tensor) -> torch.Tensor:
    """[B, h, S, D] -> [B * S, h, D] (a view where the strides allow it)."""
    B, h, S, D = t.shape
    return t.transpose(1, 2).reshape(B * S, h, D)


def _epilogue_kv8_batch(q, k, v, cache: PagedKVCache8, positions, rope_theta, qn, kn, eps, rope_table, out):
    """qkv_epilogue of [B, h, S, D] tensors into an 8-bit cache whose blocks are reserved, from its present
    device lengths on; `out` [B * S, H, D] takes Q."""
    B, H, S, D = q.shape
    pos = table = None
    if rope_table is not None:
        table = tuple(t.to(torch.float32) for t in rope_table)
        if table[0].shape[0] != B * S:
            table = tuple(t.repeat(B, 1) for t in table)
        table = tuple(t.contiguous() for t in table)
    else:
        pos = positions.to(torch.int64)
        if pos.numel() == B * S:
            pos = pos.reshape(-1).contiguous()
        else:
            pos = (pos.reshape(1, -1) if pos.dim() < 2 else pos).expand(B, S).reshape(-1).contiguous()   # of one position reshape makes a view
    cu = cache.one_each[:B + 1] if S == 1 else torch.arange(0, B * S + 1, S, dtype=torch.int32, device=q.device)
    qkv_epilogue_kv8(_flat_tokens(q), _flat_tokens(k), _flat_tokens(v), cache, cu, cache.lengths[:B], pos, rope_theta,
                     table, qn, kn, eps, out)


def _prefill_kv8(q: torch.Tensor, cache: PagedKVCache8, cu_dev: torch.Tensor, B: int, max_q: int, num_kv_heads: int):
    """Causal attention of packed Q [H, T, D] over an 8-bit cache: the sequences' rows are read back (exactly) into
    bf16 staging and go through the varlen prefill kernel, so a row sees the values every later step sees."""
    H, T, D = q.shape
    out = torch.empty((T, H * D), dtype=BF16, device=q.device)
    if T == 0:
        return out
    lens = cache.lengths[:B]
    rows = max(cache.host_lengths()[:B])
    kst, vst = kv8_read(cache, lens, rows)
    _launch(q.get_device(), "mllm_prefill_attention_varlen_bf16", _ptr(q), _ptr(kst), _ptr(vst), num_kv_heads * rows * D,
            rows * D, D, rows, _ptr(cu_dev), _ptr(lens), B, H, num_kv_heads, D, T, max_q, 1.0 / math.sqrt(D), _ptr(out))
    return out


def qkv_epilogue(q, k, v, kv_cache: KVCache, positions: torch.Tensor, rope_theta: float,
                 q_norm_weight=None, k_norm_weight=None, eps: float = 1e-6,
                 rope_table=None) -> torch.Tensor:
    """Fused per-head QK-RMSNorm (optional) + RoPE + KV append.  q [B,H,S,D], k/v [B,Hkv,S,D]
    as strided views of the projections; positions int64 [S] (shared) or [B, S].  Rows go to
    cache slots lengths[b] + s; the cache lengths advance by S.  Returns Q [B,H,S,D] (rotated)."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        _check_cuda_bf16(n, t)
        if t.dim() != 4 or t.stride(3) != 1:
            raise RuntimeError(f"Attention: {n} must be rank-4 [B, h, S, D] with D contiguous")
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if H % Hkv != 0:
        raise RuntimeError("Attention: num_heads must be divisible by num_kv_heads.")
    if isinstance(kv_cache, PagedKVCache8):
        for b in range(B):
            kv_cache.reserve(b, kv_cache.host_lengths()[b] + S)
        packed = torch.empty((H, B * S, D), dtype=BF16, device=q.device)   # the layout the packed prefill reads
        _epilogue_kv8_batch(q, k, v, kv_cache, positions, rope_theta, q_norm_weight, k_norm_weight, eps, rope_table,
                            packed.transpose(0, 1))
        kv_cache.advance(S, batch=B)
        return packed.view(H, B, S, D).transpose(0, 1)
    q_out = torch.empty((B, H, S, D), dtype=BF16, device=q.device)
    pos = positions.to(torch.int64)
    if pos.dim() == 1:
        pos_sb, pos_ss = 0, pos.stride(0)
    else:
        pos_sb, pos_ss = pos.stride(0), pos.stride(1)
    cos = sin = None
    rsb = rss = 0
    if rope_table is not None:
        cos, sin = (t.to(torch.float32).contiguous() for t in rope_table)
        rsb, rss = (0, 1) if cos.shape[0] == S else (S, 1)
    qn = kn = None
    if q_norm_weight is not None:
        qn = q_norm_weight.to(BF16).contiguous()
        kn = k_norm_weight.to(BF16).contiguous()
    if isinstance(kv_cache, PagedKVCache):
        start = kv_cache.lengths[:B].clone()   # slots of the new rows: the lengths before this call
        for b in range(B):
            kv_cache.reserve(b, kv_cache.host_lengths()[b] + S)
        kv = kv_cache.descriptor()
        abi.call("mllm_qkv_epilogue_paged_bf16",
                 _ptr(q), q.stride(0), q.stride(2), q.stride(1),
                 _ptr(k), k.stride(0), k.stride(2), k.stride(1),
                 _ptr(v), v.stride(0), v.stride(2), v.stride(1),
                 B, S, H, Hkv, D, _ptr(pos), pos_sb, pos_ss, float(rope_theta),
                 _ptr(cos), _ptr(sin), rsb, rss, _ptr(qn), _ptr(kn), float(eps), _ptr(q_out),
                 C.byref(kv), _ptr(start), 0, abi.stream_handle())
        kv_cache.advance(S, batch=B)
        return q_out
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_qkv_epilogue_bf16",
             _ptr(q), q.stride(0), q.stride(2), q.stride(1),
             _ptr(k), k.stride(0), k.stride(2), k.stride(1),
             _ptr(v), v.stride(0), v.stride(2), v.stride(1),
             B, S, H, Hkv, D, _ptr(pos), pos_sb, pos_ss, float(rope_theta),
             _ptr(cos), _ptr(sin), rsb, rss, _ptr(qn), _ptr(kn), float(eps), _ptr(q_out),
             _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf), csb, csh, cst, kv_cache.capacity,
             _ptr(kv_cache.lengths), 0, abi.stream_handle())
    kv_cache.advance(S)
    return q_out


def prefill_attention(q: torch.Tensor, kv_cache: KVCache, num_kv_heads: int) -> torch.Tensor:
    """Causal attention of Q [B,H,S,D] (the newest S rows) over the cache -> [B, S, H*D]."""
    B, H, S, D = q.shape
    if isinstance(kv_cache, PagedKVCache8):
        cu = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=q.device) if S else None
        packed = q.transpose(0, 1).reshape(H, B * S, D)
        return _prefill_kv8(packed, kv_cache, cu, B, S, num_kv_heads).view(B, S, H * D)
    out = torch.empty((B, S, H * D), dtype=BF16, device=q.device)
    if isinstance(kv_cache, PagedKVCache):
        kv = kv_cache.descriptor()
        abi.call("mllm_prefill_attention_paged_bf16", _ptr(q), C.byref(kv), B, H, num_kv_heads, D, S,
                 kv_cache.length_of(B), 1.0 / math.sqrt(D), _ptr(out), abi.stream_handle())
        return out
    kv_len = kv_cache.length
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_prefill_attention_bf16", _ptr(q), _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf),
             csb, csh, cst, B, H, num_kv_heads, D, S, kv_len, 1.0 / math.sqrt(D), _ptr(out),
             abi.stream_handle())
    return out


def _cu_seqlens(q_lens: list[int], device) -> tuple[list[int], torch.Tensor]:
    """Row offsets of packed sequences: host list and int32 device tensor [len(q_lens) + 1]."""
    if any(n < 0 for n in q_lens):
        raise RuntimeError("packed sequences: lengths must be >= 0")
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return cu, torch.tensor(cu, dtype=torch.int32).to(device, non_blocking=True)


def qkv_epilogue_packed(q, k, v, kv_cache, q_lens: list[int], rope_theta: float, positions=None,
                        q_norm_weight=None, k_norm_weight=None, eps: float = 1e-6) -> torch.Tensor:
    """qkv_epilogue (TransformerBlock.h:103-107,130-134 and Attention.h:157-208) for several
    sequences of different lengths packed on one token axis, in one launch; the reference runs one
    sequence's prompt per Generate call (QwenRunner.cpp:420-545).  q [T, H, D] and k/v [T, Hkv, D] (strided views of the projections, D contiguous);
    sequence b owns the next q_lens[b] tokens, which go to cache slots lengths[b] + s of cache
    sequence b; the lengths advance by q_lens[b].  positions: int64 [T] (default: each token's
    cache slot).  Returns Q [H, T, D] (rotated), the layout prefill_attention_packed reads."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        _check_cuda_bf16(n, t)
        if t.dim() != 3 or t.stride(2) != 1:
            raise RuntimeError(f"Attention: {n} must be rank-3 [T, h, D] with D contiguous")
    T, H, D = q.shape
    Hkv = k.shape[1]
    if H % Hkv != 0:
        raise RuntimeError("Attention: num_heads must be divisible by num_kv_heads.")
    B = len(q_lens)
    cu, cu_dev = _cu_seqlens(q_lens, q.device)
    if cu[-1] != T:
        raise RuntimeError("packed sequences: q_lens must sum to the token count")
    if T == 0:
        return torch.empty((H, 0, D), dtype=BF16, device=q.device)
    before = kv_cache.host_lengths()[:B]
    if positions is None:
        positions = torch.cat([torch.arange(before[b], before[b] + q_lens[b], dtype=torch.int64)
                               for b in range(B)]).to(q.device, non_blocking=True)
    pos = positions.to(device=q.device, dtype=torch.int64).contiguous()
    if pos.numel() != T:
        raise RuntimeError("packed sequences: one position per token")
    if isinstance(kv_cache, PagedKVCache8):
        for b in range(B):
            kv_cache.reserve(b, before[b] + q_lens[b])
        q_out = torch.empty((H, T, D), dtype=BF16, device=q.device)
        qkv_epilogue_kv8(q, k, v, kv_cache, cu_dev, kv_cache.lengths[:B], pos.reshape(-1), rope_theta, None, q_norm_weight,
                         k_norm_weight, eps, q_out.transpose(0, 1))
        kv_cache.advance(list(q_lens), batch=B)   # behind all that the epilogue may refuse
        return q_out
    qn = kn = None
    if q_norm_weight is not None:
        qn = q_norm_weight.to(BF16).contiguous()
        kn = k_norm_weight.to(BF16).contiguous()
    q_out = torch.empty((H, T, D), dtype=BF16, device=q.device)
    start = kv_cache.lengths[:B].clone()    # slots of the new rows: the lengths before this call
    common = (_ptr(q), q.stride(0), q.stride(1), _ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0),
              v.stride(1), T, H, Hkv, D, _ptr(pos), float(rope_theta), _ptr(qn), _ptr(kn), float(eps),
              _ptr(q_out))
    if isinstance(kv_cache, PagedKVCache):
        kv_cache.advance(list(q_lens), batch=B)   # reserves the blocks; raises before any launch
        kv = kv_cache.descriptor()
        abi.call("mllm_qkv_epilogue_varlen_paged_bf16", *common, C.byref(kv), _ptr(cu_dev), B, _ptr(start),
                 abi.stream_handle())
        return q_out
    if B != len(kv_cache.host_lengths()):
        raise RuntimeError("packed sequences: one length per cache sequence")
    kv_cache.advance(list(q_lens))                # raises before any launch if the cache is full
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_qkv_epilogue_varlen_bf16", *common, _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf), csb,
             csh, cst, kv_cache.capacity, _ptr(cu_dev), B, _ptr(start), abi.stream_handle())
    return q_out


def prefill_attention_packed(q: torch.Tensor, kv_cache, q_lens: list[int], num_kv_heads: int) -> torch.Tensor:
    """Causal attention (Attention.h:220-316) of packed sequences: Q [H, T, D]
    (qkv_epilogue_packed's output, sequence b owning the next q_lens[b] rows, its newest rows) over each sequence's cache rows
    0 .. lengths[b] - 1 -> [T, H*D]."""
    H, T, D = q.shape
    B = len(q_lens)
    cu, cu_dev = _cu_seqlens(q_lens, q.device)
    if cu[-1] != T:
        raise RuntimeError("packed sequences: q_lens must sum to the token count")
    max_q = max(q_lens) if q_lens else 0
    if isinstance(kv_cache, PagedKVCache8):
        return _prefill_kv8(q.contiguous(), kv_cache, cu_dev, B, max_q, num_kv_heads)
    out = torch.empty((T, H * D), dtype=BF16, device=q.device)
    kv_lens = kv_cache.lengths[:B]
    if isinstance(kv_cache, PagedKVCache):
        kv = kv_cache.descriptor()
        abi.call("mllm_prefill_attention_varlen_paged_bf16", _ptr(q), C.byref(kv), _ptr(cu_dev), _ptr(kv_lens), B,
                 H, num_kv_heads, D, T, max_q, 1.0 / math.sqrt(D), _ptr(out), abi.stream_handle())
        return out
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_prefill_attention_varlen_bf16", _ptr(q), _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf),
             csb, csh, cst, kv_cache.capacity, _ptr(cu_dev), _ptr(kv_lens), B, H, num_kv_heads, D, T, max_q,
             1.0 / math.sqrt(D), _ptr(out), abi.stream_handle())
    return out


def decode_attention(q: torch.Tensor, kv_cache: KVCache, num_kv_heads: int,
                     max_kv_len: int | None = None) -> torch.Tensor:
    """One query row per sequence (Q [B,H,1,D] or [B,H,D]) over each sequence's cache rows
    (per-sequence lengths) -> [B, 1, H*D]."""
    if isinstance(kv_cache, PagedKVCache8):
        return _decode_kv8(q, kv_cache, num_kv_heads, max_kv_len)
    B, H, D = q.shape[0], q.shape[1], q.shape[-1]
    qq = q.reshape(B, H, D)
    if not qq.is_contiguous():
        qq = qq.contiguous()
    L = max_kv_len or max(kv_cache.host_lengths()[:B])
    L = min(L, kv_cache.capacity)
    out = torch.empty((B, 1, H * D), dtype=BF16, device=q.device)
    lib = abi.load()
    nbytes = lib.mllm_decode_attention_workspace_size(B, H, num_kv_heads, D, L)
    ws = _capture_scratch.get("decode", nbytes, q.device) if _capturing() else _WS.get(nbytes, q.device)
    if isinstance(kv_cache, PagedKVCache):
        kv = kv_cache.descriptor()
        abi.call("mllm_decode_attention_paged_bf16", _ptr(qq), C.byref(kv), _ptr(kv_cache.lengths), B, H,
                 num_kv_heads, D, L, 1.0 / math.sqrt(D), _ptr(out), _ptr(ws), ws.numel(), abi.stream_handle())
        return out
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_decode_attention_bf16", _ptr(qq), _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf),
             csb, csh, cst, _ptr(kv_cache.lengths), B, H, num_kv_heads, D, L, 1.0 / math.sqrt(D),
             _ptr(out), _ptr(ws), ws.numel(), abi.stream_handle())
    return out


def decode_attention_shared(q: torch.Tensor, kv_cache: PagedKVCache, num_kv_heads: int, prefix_len: int,
                            max_kv_len: int | None = None) -> torch.Tensor:
    """decode_attention over a paged cache whose sequences 0 .. B-1 all begin with the same prefix_len
    rows (PagedKVCache.fork): the prefix is read once for the whole batch, through the table row of
    the first sequence that is not empty, every sequence's further rows through its own -> [B, 1, H*D].
    Lengths come from the cache (each at least prefix_len, or 0)."""
    if not isinstance(kv_cache, PagedKVCache):
        raise RuntimeError("decode_attention_shared: needs a PagedKVCache or a PagedKVCache8")
    q, (B, H, D), dev, L = _decode_args(q, kv_cache, num_kv_heads, max_kv_len)
    device = q.device
    out = torch.empty_strided((B, 1, H * D), (H * D, H * D, 1), dtype=BF16, device=device)
    nbytes = _workspace_size("mllm_decode_attention_shared_workspace_size", B, H, num_kv_heads, D, prefix_len)
    ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=device)   # of the call's own, as in _decode_kv8
    name = "mllm_decode_attention_shared_paged_kv8" if isinstance(kv_cache, PagedKVCache8) else \
        "mllm_decode_attention_shared_paged_bf16"
    _launch(dev, name, q.data_ptr(), C.byref(kv_cache.descriptor()),
            kv_cache.lengths.data_ptr(), prefix_len, B, H, num_kv_heads, D, L, 1.0 / math.sqrt(D), out.data_ptr(),
            ws.data_ptr(), nbytes)
    return out


def _decode_step_kv8(q, k, v, cache: PagedKVCache8, positions, rope_theta, num_kv_heads, qn, kn, eps, rope_table):
    """decode_step over an 8-bit cache: the epilogue appends at the device lengths, which then advance."""
    B, H, _, D = q.shape
    capturing = _capturing()
    if capturing and cache.capture_max_len is None:
        raise RuntimeError("decode_step: set the cache's capture_max_len before capturing a graph")
    if not capturing:   # raises before any launch if the pool is full
        for b in range(B):
            cache.reserve(b, cache.host_lengths()[b] + 1)
    q_rot = torch.empty((B, H, D), dtype=BF16, device=q.device)
    _epilogue_kv8_batch(q, k, v, cache, positions, rope_theta, qn, kn, eps, rope_table, q_rot)
    if capturing:
        cache.lengths[:B] += 1
        L = cache.capture_max_len
    else:
        cache.advance(1, batch=B)
        L = max(cache.host_lengths()[:B])
    L = min(L, cache.capacity)
    if cache.shared_prefix > 0 and _shared_pays(B, cache.shared_prefix, num_kv_heads, D, True) and \
            cache._rows_in_common(B, cache.shared_prefix):
        return decode_attention_shared(q_rot, cache, num_kv_heads, cache.shared_prefix, L)
    return _decode_kv8(q_rot, cache, num_kv_heads, L)


# Bytes of a prefix that reading it once has to save for the shared decode to pay for its launches: a step of 32 / 8 heads
# of 128 takes 18 us with any short prefix against 11 to 15 us fused (up to 32 MB saved), 24 against 24 at 34 MB
# (2 sequences, 8192 rows), 20 against 23 at 59 MB (8, 2048) and 51 against 236 at 2 GB (16, 32768).
_SHARED_MIN_BYTES = 40 << 20


# Of an 8-bit cache, whose rows the shared form has to convert: 20 us against 26 with 130 MB saved (32 sequences, 2048
# rows), 24 against 27 with 117 MB (8, 8192), 24 against 19 with 50 MB (4, 8192); and 52 against 45 with 200 MB for 4
# sequences behind 32700 rows, where there are too few query rows to each converted one.
_SHARED_MIN_BYTES8 = 100 << 20
_SHARED_MIN_BATCH8 = 6


def _shared_pays(B: int, prefix: int, num_kv_heads: int, D: int, kv8: bool = False) -> bool:
    rows = (B - 1) * prefix * num_kv_heads * D
    if kv8:
        return B >= _SHARED_MIN_BATCH8 and rows * 2 >= _SHARED_MIN_BYTES8
    return rows * 4 >= _SHARED_MIN_BYTES


def _check_step(q, k, v, cache: PagedKVCache, positions, num_kv_heads: int, rope_table) -> None:
    """What a step of an append and a decode of their own can refuse, before the first of them is launched."""
    B, H, _, D = q.shape
    pool = cache.k_pool.shape
    if H > 8 * num_kv_heads:
        raise RuntimeError("decode_step: GQA group larger than 8")
    if B > cache.block_table.shape[0] or pool[1] != num_kv_heads or pool[3] != D or k.shape != (B, num_kv_heads, 1, D) or \
            v.shape != k.shape:
        raise RuntimeError("decode_step: k, v and the cache must have num_kv_heads heads of q's head_dim, and a row per "
                           "sequence")
    if rope_table is not None:
        if any(tuple(t.shape) not in ((1, D), (B, D)) for t in rope_table) or rope_table[0].shape != rope_table[1].shape:
            raise RuntimeError("RoPE: tables must be [1, D] or [B, D] in a decode step")
    elif positions.numel() not in (1, B):
        raise RuntimeError("RoPE: one position, or one per sequence, in a decode step")


def _decode_step_shared(q, k, v, cache: PagedKVCache, positions, rope_theta, num_kv_heads, qn, kn, eps, rope_table):
    """decode_step over a cache whose sequences share their first rows: the epilogue appends at the device lengths,
    which then advance, and the attention reads the prefix once."""
    B, H, _, D = q.shape
    capturing = _capturing()
    if capturing and cache.capture_max_len is None:
        raise RuntimeError("decode_step: set the cache's capture_max_len before capturing a graph")
    if not capturing:   # raises before any launch if the pool is full
        for b in range(B):
            cache.reserve(b, cache.host_lengths()[b] + 1)
    pos = positions.to(torch.int64).reshape(-1)
    cos = sin = None
    rsb = 0
    if rope_table is not None:
        cos, sin = (t.to(torch.float32).contiguous() for t in rope_table)
        rsb = 0 if cos.shape[0] == 1 else 1
    if qn is not None:
        qn, kn = qn.to(BF16).contiguous(), kn.to(BF16).contiguous()
    q_rot = torch.empty((B, H, D), dtype=BF16, device=q.device)
    kv = cache.descriptor()
    _launch(q.get_device(), "mllm_qkv_epilogue_paged_bf16", _ptr(q), q.stride(0), q.stride(2), q.stride(1), _ptr(k),
            k.stride(0), k.stride(2), k.stride(1), _ptr(v), v.stride(0), v.stride(2), v.stride(1), B, 1, H, num_kv_heads, D,
            _ptr(pos), 0 if pos.numel() == 1 else pos.stride(0), 0, float(rope_theta), _ptr(cos), _ptr(sin), rsb, 0,
            _ptr(qn), _ptr(kn), float(eps), _ptr(q_rot), C.byref(kv), _ptr(cache.lengths), 0)
    if capturing:
        cache.lengths[:B] += 1
        L = cache.capture_max_len
    else:
        cache.advance(1, batch=B)
        L = max(cache.host_lengths()[:B])
    return decode_attention_shared(q_rot, cache, num_kv_heads, cache.shared_prefix, min(L, cache.capacity))


def decode_step(q, k, v, kv_cache: KVCache, positions: torch.Tensor, rope_theta: float, num_kv_heads: int,
                q_norm_weight=None, k_norm_weight=None, eps: float = 1e-6, rope_table=None) -> torch.Tensor:
    """One new token per sequence through the fused step: QK-RMSNorm (optional) + RoPE + KV
    append + decode attention in one launch.  q [B,H,1,D], k/v [B,Hkv,1,D] (strided views of the
    projections); positions int64 [1] (shared) or [B] / [B, 1].  The new rows go to slot
    lengths[b] of each sequence and the lengths advance by one.  Returns [B, 1, H*D].  A paged cache
    whose shared_prefix is set is read by decode_attention_shared, after an epilogue launch of its own,
    where the sequences came by that many rows together (PagedKVCache.fork) and batch and prefix are
    large enough for that to be faster; else each sequence's rows are read through its own table row."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        _check_cuda_bf16(n, t)
        if t.dim() != 4 or t.size(2) != 1 or t.stride(3) != 1:
            raise RuntimeError(f"Attention: {n} must be [B, h, 1, D] with D contiguous")
    B, H, _, D = q.shape
    if H % num_kv_heads != 0:
        raise RuntimeError("Attention: num_heads must be divisible by num_kv_heads.")
    if isinstance(kv_cache, PagedKVCache8):
        _check_step(q, k, v, kv_cache, positions, num_kv_heads, rope_table)
        return _decode_step_kv8(q, k, v, kv_cache, positions, rope_theta, num_kv_heads, q_norm_weight, k_norm_weight,
                                eps, rope_table)
    if isinstance(kv_cache, PagedKVCache) and kv_cache.shared_prefix > 0:
        _check_step(q, k, v, kv_cache, positions, num_kv_heads, rope_table)
        if _shared_pays(B, kv_cache.shared_prefix, num_kv_heads, D) and \
                kv_cache._rows_in_common(B, kv_cache.shared_prefix):
            return _decode_step_shared(q, k, v, kv_cache, positions, rope_theta, num_kv_heads, q_norm_weight,
                                       k_norm_weight, eps, rope_table)
    pos = positions.to(torch.int64).reshape(-1)
    pos_sb = 0 if pos.numel() == 1 else pos.stride(0)
    cos = sin = None
    rsb = 0
    if rope_table is not None:
        cos, sin = (t.to(torch.float32).contiguous() for t in rope_table)
        rsb = 0 if cos.shape[0] == 1 else 1
    qn = kn = None
    if q_norm_weight is not None:
        qn = q_norm_weight.to(BF16).contiguous()
        kn = k_norm_weight.to(BF16).contiguous()
    capturing = _capturing()
    if capturing:
        # Recorded into a CUDA graph that replays this step many times: the lengths advance on the
        # device (the caller advances the host copy after each replay, and reserved the blocks
        # beforehand), and the bound on every sequence's length is the one the graph was made for.
        if kv_cache.capture_max_len is None:
            raise RuntimeError("decode_step: set the cache's capture_max_len before capturing a graph")
        kv_cache.lengths[:B] += 1
        L = min(kv_cache.capture_max_len, kv_cache.capacity)
    else:
        if isinstance(kv_cache, PagedKVCache):
            kv_cache.advance(1, batch=B)   # reserves the blocks; raises before any launch if the pool is full
        else:
            kv_cache.advance(1)   # raises before any launch if the cache is full
        L = min(max(kv_cache.host_lengths()[:B]), kv_cache.capacity)
    out = torch.empty((B, 1, H * D), dtype=BF16, device=q.device)
    lib = abi.load()
    nbytes = lib.mllm_decode_attention_workspace_size(B, H, num_kv_heads, D, L)
    ws = _capture_scratch.get("decode", nbytes, q.device) if capturing else _WS.get(nbytes, q.device)
    if isinstance(kv_cache, PagedKVCache):
        kv = kv_cache.descriptor()
        abi.call("mllm_decode_step_paged_bf16",
                 _ptr(q), q.stride(0), q.stride(1), _ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0),
                 v.stride(1), _ptr(pos), pos_sb, float(rope_theta), _ptr(cos), _ptr(sin), rsb, _ptr(qn), _ptr(kn),
                 float(eps), C.byref(kv), _ptr(kv_cache.lengths), B, H, num_kv_heads, D, L, 1.0 / math.sqrt(D),
                 _ptr(out), _ptr(ws), ws.numel(), abi.stream_handle())
        return out
    csb, csh, cst = kv_cache.strides
    abi.call("mllm_decode_step_bf16",
             _ptr(q), q.stride(0), q.stride(1), _ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0), v.stride(1),
             _ptr(pos), pos_sb, float(rope_theta), _ptr(cos), _ptr(sin), rsb, _ptr(qn), _ptr(kn), float(eps),
             _ptr(kv_cache.key_buf), _ptr(kv_cache.value_buf), csb, csh, cst, _ptr(kv_cache.lengths),
             B, H, num_kv_heads, D, L, 1.0 / math.sqrt(D), _ptr(out), _ptr(ws), ws.numel(), abi.stream_handle())
    return out


def _rows(name: str, t: torch.Tensor, B: int, dtype, dev: int):
    """A [B, n] tensor on device number `dev` whose rows are contiguous, or a copy of it where the rows overlap (an
    expanded one): (the tensor, its row stride, n).  The stride of a single row means nothing."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != B or t.dtype is not dtype or t.get_device() != dev or \
            (shape[1] > 1 and stride[1] != 1):
        raise RuntimeError(f"{name}: expected a {dtype} [{B}, n] tensor with contiguous rows on cuda:{dev}")
    n = shape[1]
    if stride[0] >= n:
        return t, stride[0], n
    return t if B < 2 else t.contiguous(), n, n


MAX_LOGIT_BIASES = 1024


def apply_logit_rules(logits: torch.Tensor, history=None, history_lens=None, output_start=None, repetition=None,
                      presence=None, frequency=None, bias_ids=None, bias_values=None, bias_lens=None, allowed=None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and a mask of allowed tokens on logits [B, V] bf16 or fp32 (mllm_logit_rules),
    each row with its own, before `sample`:
      history int64 [B, n] with history_lens int32 [B]: the row's tokens, prompt first; those from
        output_start int32 [B] (default 0) on are generated ones
      repetition, presence, frequency fp32 [B]: a seen token's logit is divided by the first (multiplied
        where negative), a generated token's lowered by the second, and by the third for each time
      bias_ids int64 / bias_values fp32 [B, n <= 1024] with bias_lens int32 [B]: added to tokens
      allowed int32 [B, ceil(V / 32)]: bit v % 32 of word v // 32 allows token v; others become -inf
    All on the device.  Returns `out` (a new tensor by default; `logits` itself works in place, another
    view of its rows is refused)."""
    if not logits.is_cuda:
        raise RuntimeError("logit rules: logits must be a CUDA tensor (no CPU fallback)")
    dtype = logits.dtype
    if dtype is not BF16 and dtype is not torch.float32:
        raise RuntimeError("logit rules: logits must be bf16 or fp32")
    if logits.dim() != 2:
        raise RuntimeError("logit rules: logits must be [B, V]")
    B, V = shape = logits.shape
    dev = logits.get_device()
    logits, x_stride, _ = _rows("logits", logits, B, dtype, dev)
    if (history is None) != (history_lens is None):
        raise RuntimeError("logit rules: give both history and history_lens or neither")
    hist_stride = hist_cols = bias_stride = bias_cols = words_stride = 0
    if history is not None:
        history, hist_stride, hist_cols = _rows("history", history, B, torch.int64, dev)
        _check_vec("history_lens", history_lens, B, torch.int32, dev)
    if output_start is not None:
        _check_vec("output_start", output_start, B, torch.int32, dev)
    if repetition is not None:
        _check_vec("repetition", repetition, B, torch.float32, dev)
    if presence is not None:
        _check_vec("presence", presence, B, torch.float32, dev)
    if frequency is not None:
        _check_vec("frequency", frequency, B, torch.float32, dev)
    if bias_ids is not None and bias_values is not None and bias_lens is not None:
        bias_ids, bias_stride, bias_cols = _rows("bias_ids", bias_ids, B, torch.int64, dev)
        bias_values, stride, n = _rows("bias_values", bias_values, B, torch.float32, dev)
        _check_vec("bias_lens", bias_lens, B, torch.int32, dev)
        if n != bias_cols:
            raise RuntimeError("logit rules: bias_ids and bias_values must have the same shape")
        if stride != bias_stride:
            bias_ids, bias_values, bias_stride = bias_ids.contiguous(), bias_values.contiguous(), n
    if allowed is not None:
        allowed, words_stride, n = _rows("allowed", allowed, B, torch.int32, dev)
        if n < (V + 31) // 32:
            raise RuntimeError("logit rules: allowed needs ceil(V / 32) words a row")
    if history is not None and hist_cols == 0:
        history = history_lens = output_start = repetition = presence = frequency = None
    if bias_ids is not None and bias_cols == 0:
        bias_ids = bias_values = bias_lens = None
    if out is None:
        out = torch.empty_strided(shape, (V, 1), dtype=dtype, device=logits.device)
        y_stride = V
    else:
        y_stride, step = out.stride() if out.dim() == 2 else (0, 0)
        if out.shape != shape or out.dtype is not dtype or out.get_device() != dev or (V > 1 and step != 1) or \
                (B > 1 and y_stride < V):
            raise RuntimeError("logit rules: out must be like logits, its rows apart")
        y_stride = max(y_stride, V)
    if B == 0 or V == 0:
        return out
    _launch(dev, "mllm_logit_rules", logits.data_ptr(), int(dtype is BF16), x_stride, B, V, _ptr(history), hist_stride,
            hist_cols, _ptr(history_lens), _ptr(output_start), _ptr(repetition), _ptr(presence), _ptr(frequency),
            _ptr(bias_ids), _ptr(bias_values), bias_stride, bias_cols, _ptr(bias_lens), _ptr(allowed), words_stride,
            out.data_ptr(), y_stride)
    return out


_SAMPLE_WS = DecodeWorkspace()


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           use_greedy: bool = False, previous_tokens=None, repetition_penalty: float = 1.0,
           seed: int = 0, offset: int = 0) -> torch.Tensor:
    """Sampler::Sample (Sampler.cpp:49-232) on the device for a batch of rows: logits [B, V] (or
    [V]) bf16 or fp32 CUDA, penalised IN PLACE like the reference; previous_tokens: a list of
    per-row token lists (or one list for a single row).  Returns the int64 token ids [B] on the
    device, without a host round trip.  The sampling draw of row b comes from Philox-4x32-10 with
    key `seed` and counter (offset, b, 0)."""
    if not logits.is_cuda:
        raise RuntimeError("Sampler: logits must be a CUDA tensor (no CPU fallback)")
    if logits.dtype not in (BF16, torch.float32):
        raise RuntimeError("Sampler: logits must be bf16 or fp32")
    x = logits if logits.dim() == 2 else logits.view(1, -1)
    if x.stride(1) != 1:
        raise RuntimeError("Sampler: logits rows must be contiguous")
    B, V = x.shape
    prev = cnt = None
    if previous_tokens is not None:
        rows = previous_tokens if (len(previous_tokens) and isinstance(previous_tokens[0], (list, tuple))) \
            else [previous_tokens]
        if len(rows) != B:
            raise RuntimeError("Sampler: one history per row")
        T = max(1, max(len(r) for r in rows))
        h = torch.full((B, T), -1, dtype=torch.int64)
        for b, r in enumerate(rows):
            h[b, : len(r)] = torch.tensor(list(r), dtype=torch.int64)
        prev = h.to(x.device, non_blocking=True)
        cnt = torch.tensor([len(r) for r in rows], dtype=torch.int32).to(x.device, non_blocking=True)
    out = torch.empty(B, dtype=torch.int64, device=x.device)
    lib = abi.load()
    ws = _SAMPLE_WS.get(lib.mllm_sample_workspace_size(B, V), x.device)
    abi.call("mllm_sample", _ptr(x), int(x.dtype == BF16), x.stride(0), B, V, _ptr(prev),
             prev.stride(0) if prev is not None else 0, _ptr(cnt), float(temperature), int(top_k), float(top_p),
             int(bool(use_greedy)), float(repetition_penalty), int(seed), int(offset), _ptr(out), _ptr(ws),
             ws.numel(), abi.stream_handle())
    return out


LINEAR_MAX_TOKENS = 256


def linear_supported(x: torch.Tensor, weights) -> bool:
    """Whether mllm_linear_bf16 takes this projection: bf16 CUDA tensors, at most 256 rows of x,
    K a multiple of 64, each weight's rows a multiple of 128, unit inner strides."""
    if not (x.is_cuda and x.dtype == BF16 and x.stride(-1) == 1 and 0 < len(weights) <= 4):
        return False
    T = x.numel() // x.size(-1) if x.size(-1) else 0
    K = x.size(-1)
    if T > LINEAR_MAX_TOKENS or K % 64 != 0:
        return False
    return all(w.is_cuda and w.dtype == BF16 and w.dim() == 2 and w.size(1) == K and w.stride(1) == 1
               and w.size(0) % 128 == 0 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0 for w in weights)


def linear(x: torch.Tensor, weights) -> torch.Tensor:
    """Linear::Forward (Linear.h:33-68) of up to four weights in one launch (mllm_linear_bf16):
    x [..., K] bf16 with at most 256 rows -> [..., sum of out_features], the weights' outputs
    side by side (q | k | v for the three attention projections).  fp32 accumulation, one
    rounding to bf16."""
    weights = list(weights)
    if not linear_supported(x, weights):
        raise RuntimeError("linear: needs bf16 CUDA tensors, <= 256 rows, K % 64 == 0, weight rows % 128 == 0")
    lead = x.shape[:-1]
    K = x.size(-1)
    x2 = x.reshape(-1, K)
    if x2.stride(0) % 8 != 0 or x2.data_ptr() % 16 != 0:
        x2 = x2.contiguous()
    T = x2.size(0)
    n = [w.size(0) for w in weights]
    out = torch.empty((T, sum(n)), dtype=BF16, device=x.device)
    W = len(weights)
    wp = (C.c_void_p * W)(*[w.data_ptr() for w in weights])
    wst = (C.c_int64 * W)(*[w.stride(0) for w in weights])
    nf = (C.c_int64 * W)(*n)
    need = abi.load().mllm_linear_workspace_size(T, W, nf, K)
    if need and _capturing():
        ws = _capture_scratch.get("linear", need, x.device)
    else:
        ws = _linear_workspace(x.device, need)
    abi.call("mllm_linear_bf16", _ptr(x2), x2.stride(0), T, K, W, wp, wst, nf, _ptr(out), out.stride(0),
             _ptr(ws), ws.numel() if ws is not None else 0, abi.stream_handle())
    return out.view(*lead, sum(n))


_LINEAR_WS: dict = {}


def _linear_workspace(device, nbytes: int):
    """The split partials and tile counters of mllm_linear_bf16: one zero-filled buffer per
    (device, stream), grown on demand; every call leaves its counters at zero."""
    if nbytes == 0:
        return None
    key = (device, torch.cuda.current_stream(device).cuda_stream)
    ws = _LINEAR_WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _LINEAR_WS[key] = ws
    return ws


class Fp8Weight:
    """A projection stored the way FP8 checkpoints hold it (QwenRunner.cpp:148-283 loads it with its
    `weight_scale_inv`): e4m3 values w [out, in] and fp32 scales [out/128, in/128], one per
    128 x 128 block.  The reference dequantizes it on every step (DequantizeFP8,
    QwenRunner.cpp:103-122) and multiplies in bf16; `linear_fp8` multiplies it as stored."""

    BLOCK = 128

    def __init__(self, w: torch.Tensor, scale_inv: torch.Tensor):
        if w.dtype != torch.float8_e4m3fn or w.dim() != 2:
            raise RuntimeError("Fp8Weight: e4m3 [out, in] weights")
        n, k = w.shape
        if n % self.BLOCK or k % self.BLOCK or tuple(scale_inv.shape) != (n // self.BLOCK, k // self.BLOCK):
            raise RuntimeError("Fp8Weight: 128 x 128 blocks, scales [out/128, in/128]")
        self.w = w.contiguous()
        self.scale_inv = scale_inv.float().contiguous()

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Fp8Weight":
        """Block-wise e4m3 quantization of a weight (scale = block amax / 448), the format of
        FP8 checkpoints; for building test and benchmark models."""
        n, k = w.shape
        b = cls.BLOCK
        blocks = w.float().view(n // b, b, k // b, b)
        amax = blocks.abs().amax(dim=(1, 3)).clamp_min(1e-12)
        scale = amax / 448.0
        q = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(n, k)
        return cls(q, scale)

    def size(self, dim: int) -> int:
        return self.w.size(dim)

    @property
    def shape(self):
        return self.w.shape

    def dequantize(self, dtype=BF16) -> torch.Tensor:
        """DequantizeFP8 (QwenRunner.cpp:103-122): w.to(dtype) * scale.to(dtype), block-broadcast,
        in dtype -- the weights the reference's GEMM sees."""
        n, k = self.w.shape
        b = self.BLOCK
        w_h = self.w.to(dtype).reshape(n // b, b, k // b, b)
        s_h = self.scale_inv.to(dtype).unsqueeze(1).unsqueeze(3)
        return (w_h * s_h).reshape(n, k)


FP8_MAX_TOKENS = 128


def linear_fp8(x: torch.Tensor, w: Fp8Weight) -> torch.Tensor:
    """Linear::Forward(x, DequantizeFP8(w)) for bf16 x with at most 128 rows, by
    mllm_linear_fp8_bf16: the fp8 bytes are streamed and dequantized on chip (into tensor memory) with the
    reference's rounding, so the product equals a bf16 GEMM on the dequantized weight (fp32
    accumulation, one rounding).  More rows: the reference's own route (dequantize, cuBLAS)."""
    K = x.size(-1)
    if K != w.size(1):
        raise RuntimeError("Linear: last dim of x must match weight in_features.")
    lead = x.shape[:-1]
    x2 = x.reshape(-1, K)
    T = x2.size(0)
    if not (x.is_cuda and x.dtype == BF16) or T > FP8_MAX_TOKENS:
        return torch.nn.functional.linear(x, w.dequantize(x.dtype))
    if x2.stride(-1) != 1 or x2.stride(0) % 8 != 0 or x2.data_ptr() % 16 != 0:
        x2 = x2.contiguous()
    N = w.size(0)
    out = torch.empty((T, N), dtype=BF16, device=x.device)
    need = abi.load().mllm_linear_fp8_workspace_size(T, N, K)
    if need and _capturing():
        ws = _capture_scratch.get("linear", need, x.device)
    else:
        ws = _linear_workspace(x.device, need)
    abi.call("mllm_linear_fp8_bf16", _ptr(x2), x2.stride(0), T, K, _ptr(w.w), w.w.stride(0), N, _ptr(w.scale_inv),
             w.scale_inv.stride(0), _ptr(out), out.stride(0), _ptr(ws), ws.numel() if ws is not None else 0,
             abi.stream_handle())
    return out.view(*lead, N)


def _linear(x: torch.Tensor, w) -> torch.Tensor:
    """Linear::Forward (Linear.h:33-68): x @ w.T in the input dtype, a cuBLAS GEMM as in the
    reference (for one weight mllm_linear_bf16 is not faster than cuBLAS beyond a few tokens);
    an Fp8Weight goes through linear_fp8."""
    if isinstance(w, Fp8Weight):
        return linear_fp8(x, w)
    if x.size(-1) != w.size(1):
        raise RuntimeError("Linear: last dim of x must match weight in_features.")
    return torch.nn.functional.linear(x, w)


def _project_qkv(h: torch.Tensor, w_q, w_k, w_v, num_heads: int, num_kv_heads: int, head_dim: int):
    """The three attention projections (TransformerBlock.h:82-96, Attention.h:52-54) as q [B,H,S,D]
    and k/v [B,Hkv,S,D] views.  Up to 256 tokens: one mllm_linear_bf16 launch writes q | k | v side
    by side and the views point into it; otherwise three cuBLAS GEMMs as in the reference (FP8
    weights: three linear_fp8 launches)."""
    B, S, E = h.shape
    if not any(isinstance(w, Fp8Weight) for w in (w_q, w_k, w_v)) and linear_supported(h, [w_q, w_k, w_v]):
        qkv = linear(h, [w_q, w_k, w_v])          # [B, S, (H + 2 Hkv) D]
        hq, hk = num_heads * head_dim, num_kv_heads * head_dim
        q = qkv[..., :hq].view(B, S, num_heads, head_dim).transpose(1, 2)
        k = qkv[..., hq:hq + hk].view(B, S, num_kv_heads, head_dim).transpose(1, 2)
        v = qkv[..., hq + hk:hq + 2 * hk].view(B, S, num_kv_heads, head_dim).transpose(1, 2)
        return q, k, v
    q = _linear(h, w_q).view(B, S, num_heads, head_dim).transpose(1, 2)
    k = _linear(h, w_k).view(B, S, num_kv_heads, head_dim).transpose(1, 2)
    v = _linear(h, w_v).view(B, S, num_kv_heads, head_dim).transpose(1, 2)
    return q, k, v


class Attention:
    @staticmethod
    def forward_projected(q, k, v, w_o, num_heads: int, num_kv_heads: int, head_dim: int,
                          rope_theta: float, position_ids: torch.Tensor, kv_cache: KVCache | None,
                          q_norm_weight=None, k_norm_weight=None, rms_norm_eps: float = 1e-6):
        """Attention::ForwardProjected (Attention.h:100-326).  q [B,H,S,D], k/v [B,Hkv,S,D]
        (views of the projections).  With norm weights, the per-head QK-RMSNorm that the
        reference runs in TransformerBlock.h:103-134 is fused into the epilogue."""
        if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
            raise RuntimeError("Attention::ForwardProjected: q/k/v must be rank-4 tensors.")
        if num_heads % num_kv_heads != 0:
            raise RuntimeError("Attention: num_heads must be divisible by num_kv_heads.")
        B, _, S, D = q.shape
        cache = kv_cache
        if cache is None:  # no cache: attend over this call's rows only (Attention.h:183 skipped)
            cache = KVCache(B, num_kv_heads, D, S, device=q.device)
        pos = position_ids.to(device=q.device)
        if S == 1:   # decode: epilogue and attention fused in one launch
            out = decode_step(q, k, v, cache, pos, rope_theta, num_kv_heads, q_norm_weight, k_norm_weight,
                              rms_norm_eps)
        else:
            qr = qkv_epilogue(q, k, v, cache, pos, rope_theta, q_norm_weight, k_norm_weight, rms_norm_eps)
            out = prefill_attention(qr, cache, num_kv_heads)
        return out if w_o is None else _linear(out, w_o)   # w_o None: the unprojected [B, S, H*D]

    @staticmethod
    def forward(hidden, w_q, w_k, w_v, w_o, num_heads: int, num_kv_heads: int, head_dim: int,
                rope_theta: float, position_ids: torch.Tensor, kv_cache: KVCache | None):
        """Attention::Forward (Attention.h:29-86): project, view, transpose, then the above."""
        if hidden.dim() != 3:
            raise RuntimeError("Attention: hidden must be [B, S, H].")
        q, k, v = _project_qkv(hidden, w_q, w_k, w_v, num_heads, num_kv_heads, head_dim)
        return Attention.forward_projected(q, k, v, w_o, num_heads, num_kv_heads, head_dim,
                                           rope_theta, position_ids, kv_cache)


def attention_block_packed(h, w_q, w_k, w_v, w_o, num_heads: int, num_kv_heads: int, head_dim: int,
                           rope_theta: float, q_lens: list[int], kv_cache, w_q_norm=None, w_k_norm=None,
                           rms_norm_eps: float = 1e-6, positions=None):
    """attention_block (TransformerBlock.h:77-195, attention half) for several prompts (or prompt
    chunks) of different lengths in one pass:
    h [T, hidden] holds the sequences' new rows back to back, sequence b the next q_lens[b] rows,
    appended to cache sequence b.  One projection, one epilogue and one attention launch for all
    of them; returns the o_proj output [T, hidden] (or [T, H*D] with w_o None)."""
    if h.dim() != 2:
        raise RuntimeError("attention_block_packed: h must be [T, hidden]")
    q, k, v = _project_qkv(h.unsqueeze(0), w_q, w_k, w_v, num_heads, num_kv_heads, head_dim)
    qr = qkv_epilogue_packed(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), kv_cache, q_lens,
                             rope_theta, positions, w_q_norm, w_k_norm, rms_norm_eps)
    out = prefill_attention_packed(qr, kv_cache, q_lens, num_kv_heads)
    return out if w_o is None else _linear(out, w_o)


def attention_block(h, w_q, w_k, w_v, w_o, num_heads: int, num_kv_heads: int, head_dim: int,
                    rope_theta: float, position_ids, kv_cache, w_q_norm=None, w_k_norm=None,
                    rms_norm_eps: float = 1e-6):
    """The attention half of TransformerBlock::Forward (TransformerBlock.h:77-195) after the
    input RMSNorm: Qwen3 branch when norm weights are given, Llama branch otherwise."""
    q, k, v = _project_qkv(h, w_q, w_k, w_v, num_heads, num_kv_heads, head_dim)
    return Attention.forward_projected(q, k, v, w_o, num_heads, num_kv_heads, head_dim, rope_theta,
                                       position_ids, kv_cache, w_q_norm, w_k_norm, rms_norm_eps)
