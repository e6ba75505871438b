"""Paged 8-bit KV cache: container, block metadata and Quest-style sparse decode.

No counterpart in the reference, whose caches are unpaged fp16 tensors; the layout is
code pools ``[num_pages, Hkv, page_size, D]`` (int8 or float8_e4m3fn), fp32 scale pools
``[num_pages, Hkv, page_size]`` and an int32 ``page_table [B, max_pages]``.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from . import _C, _lib, _workspace


@dataclass
class PagedKV:
    k_pool: Tensor
    v_pool: Tensor
    k_scale: Tensor
    v_scale: Tensor
    page_table: Tensor | None   # int32 [B, max_pages]; None: sequence b owns pages b*max_pages ...
    seq_lens: Tensor | None     # int32 [B]
    batch: int
    v_bits: int = 8             # 4: mixed-precision page records, v_pool is uint8 [num_pages, Hkv, 16, 64] (see mixed_views)

    @property
    def page_size(self) -> int:
        return self.k_pool.shape[2]

    @property
    def max_pages(self) -> int:
        return self.page_table.shape[1] if self.page_table is not None else self.k_pool.shape[0] // self.batch

    @property
    def capacity(self) -> int:
        return self.max_pages * self.page_size

    @classmethod
    def from_fused(cls, buf: Tensor, code_dtype: torch.dtype, page_table: Tensor | None, seq_lens: Tensor | None,
                   batch: int) -> "PagedKV":
        """Cache whose pools are views of one fused page-record buffer (see ``fused_views``)."""
        k, v, ks, vs = fused_views(buf, code_dtype)
        return cls(k, v, ks, vs, page_table, seq_lens, batch)

    @classmethod
    def from_mixed(cls, buf: Tensor, code_dtype: torch.dtype, page_table: Tensor | None, seq_lens: Tensor | None,
                   batch: int) -> "PagedKV":
        """Cache of mixed-precision page records: 8-bit K, 4-bit V (see ``mixed_views``)."""
        k, v, ks, vs = mixed_views(buf, code_dtype)
        return cls(k, v, ks, vs, page_table, seq_lens, batch, v_bits=4)

    def decode(self, Q: Tensor, scale: float, max_seq_len: int | None = None, out: Tensor | None = None) -> Tensor:
        """Dense GQA decode over the whole cache (``_C.fused_gqa_paged``)."""
        return _C.fused_gqa_paged(Q, self.k_pool, self.v_pool, self.k_scale, self.v_scale, self.page_table,
                                  self.seq_lens, scale, max_seq_len=max_seq_len, out=out, v_bits=self.v_bits)


RECORD_ROWS = 33  # rows of 128 bytes per (page, head): 16 of K codes, 16 of V codes, 1 of 16 + 16 fp32 scales


def fused_views(buf: Tensor, code_dtype: torch.dtype):
    """Views ``(k_pool, v_pool, k_scale, v_scale)`` over a fused page-record buffer.

    ``buf`` is uint8 ``[num_pages, Hkv, 33, 128]``: for every (page, head) the 16 K rows, the 16 V rows
    and one row holding the 16 K scales then the 16 V scales (fp32) are contiguous, so the decode kernel
    fetches a 16-token chunk with a single TMA request instead of four.  The views have the shapes every
    entry point expects (``[num_pages,Hkv,16,128]`` codes, ``[num_pages,Hkv,16]`` scales).
    """
    _C._require(buf.dtype == torch.uint8 and buf.dim() == 4 and buf.shape[2:] == (RECORD_ROWS, 128) and buf.is_contiguous(),
                "fused buffer must be contiguous uint8 [num_pages, Hkv, 33, 128]")
    k = buf[:, :, 0:16, :].view(code_dtype)
    v = buf[:, :, 16:32, :].view(code_dtype)
    sc = buf[:, :, 32, :].view(torch.float32)  # [num_pages, Hkv, 32]
    return k, v, sc[:, :, 0:16], sc[:, :, 16:32]


def pack_fused(k_pool: Tensor, v_pool: Tensor, k_scale: Tensor, v_scale: Tensor) -> Tensor:
    """Copy separate pools (page size 16, D = 128) into one fused page-record buffer."""
    num_pages, Hkv, P, D = k_pool.shape
    _C._require(P == 16 and D == 128, "fused page records need page_size 16 and head_dim 128")
    buf = torch.zeros((num_pages, Hkv, RECORD_ROWS, 128), dtype=torch.uint8, device=k_pool.device)
    k, v, ks, vs = fused_views(buf, k_pool.dtype)
    k.copy_(k_pool); v.copy_(v_pool); ks.copy_(k_scale); vs.copy_(v_scale)
    return buf


MIXED_RECORD_ROWS = 25  # 16 rows of K codes, 8 rows of 4-bit V codes (two tokens per row), 1 row of 16 + 16 fp32 scales


def mixed_views(buf: Tensor, code_dtype: torch.dtype):
    """Views ``(k_pool, v4_pool, k_scale, v_scale)`` over a buffer of mixed-precision page records.

    ``buf`` is uint8 ``[num_pages, Hkv, 25, 128]``.  K keeps 8-bit codes (``[num_pages,Hkv,16,128]`` of ``code_dtype``);
    V is stored in 4 bits, ``[num_pages,Hkv,16,64]`` uint8 with channel ``2j`` in the low and ``2j+1`` in the high
    nibble of byte ``j`` (nibble = code + 8, code in -7..7, scale = amax / 7): 200 bytes per token and head instead of
    264.  The decode kernel fetches a record with one TMA request and unpacks V in registers.
    """
    _C._require(buf.dtype == torch.uint8 and buf.dim() == 4 and buf.shape[2:] == (MIXED_RECORD_ROWS, 128) and buf.is_contiguous(),
                "mixed-precision buffer must be contiguous uint8 [num_pages, Hkv, 25, 128]")
    num_pages, Hkv = buf.shape[:2]
    k = buf[:, :, 0:16, :].view(code_dtype)
    v = buf[:, :, 16:24, :].unflatten(-1, (2, 64)).flatten(2, 3)   # [num_pages, Hkv, 16, 64]: token t = row t // 2, half t % 2
    sc = buf[:, :, 24, :].view(torch.float32)
    return k, v, sc[:, :, 0:16], sc[:, :, 16:32]


def pack_mixed(k_pool: Tensor, v4_pool: Tensor, k_scale: Tensor, v_scale: Tensor) -> Tensor:
    """Copy 8-bit K codes ``[num_pages,Hkv,16,128]``, packed 4-bit V codes ``[num_pages,Hkv,16,64]`` uint8 and their
    scales into one buffer of mixed-precision page records."""
    num_pages, Hkv, P, D = k_pool.shape
    _C._require(P == 16 and D == 128 and v4_pool.shape == (num_pages, Hkv, 16, 64) and v4_pool.dtype == torch.uint8,
                "mixed-precision records need page_size 16, head_dim 128 and uint8 [num_pages,Hkv,16,64] V codes")
    buf = torch.zeros((num_pages, Hkv, MIXED_RECORD_ROWS, 128), dtype=torch.uint8, device=k_pool.device)
    k, v, ks, vs = mixed_views(buf, k_pool.dtype)
    k.copy_(k_pool); v.copy_(v4_pool); ks.copy_(k_scale); vs.copy_(v_scale)
    return buf


def _pool_args(kv: PagedKV):
    if kv.v_bits == 4:
        kp, ks = kv.k_pool, kv.k_scale
        _C._require(kp.is_cuda and kp.dim() == 4 and kp.shape[2:] == (16, 128) and kv.v_pool.shape == (*kp.shape[:2], 16, 64)
                    and kv.v_pool.dtype == torch.uint8 and kv.v_pool.data_ptr() == kp.data_ptr() + 2048
                    and kp.stride() == (kp.shape[1] * 3200, 3200, 128, 1), "not a cache of mixed-precision page records")
        return (kp.stride(0), kp.stride(1), kp.stride(2), ks.stride(0), ks.stride(1))
    kp, ks = kv.k_pool, kv.k_scale
    _C._require(kp.is_cuda and kp.dim() == 4 and kp.stride(-1) == 1 and kv.v_pool.shape == kp.shape
                and kv.v_pool.stride() == kp.stride(), "pools must be CUDA [num_pages,Hkv,page_size,D] with one layout")
    _C._require(ks.dtype == torch.float32 and ks.shape == kp.shape[:3] and ks.stride(-1) == 1
                and kv.v_scale.stride() == ks.stride(), "scale pools must be fp32 [num_pages,Hkv,page_size]")
    return (kp.stride(0), kp.stride(1), kp.stride(2), ks.stride(0), ks.stride(1))


def build_block_meta(kv: PagedKV, block_size: int = 64, max_seq_len: int | None = None, *,
                     status: Tensor | None = None) -> Tensor:
    """Channel-wise min/max of the dequantised keys per block: fp16 ``[B, Hkv, nb, 2, D]``.

    ``status`` (optional int32 device tensor of one element) receives ``SKV_DEV_BAD_PAGE`` (2) when a page-table
    entry lies outside the pool; page 0 is read in its place."""
    strides = _pool_args(kv)
    lib = _lib.load()
    _, Hkv, P, D = kv.k_pool.shape
    N = int(max_seq_len) if max_seq_len is not None else kv.capacity
    nb = lib.skv_quest_num_blocks(N, block_size)
    meta = torch.empty((kv.batch, Hkv, nb, 2, D), dtype=torch.float16, device=kv.k_pool.device)
    dev = _C._dev_index(kv.k_pool)
    rc = lib.skv_quest_build_meta(
        kv.k_pool.data_ptr(), kv.k_scale.data_ptr(), None if kv.page_table is None else kv.page_table.data_ptr(),
        None if kv.seq_lens is None else kv.seq_lens.data_ptr(), meta.data_ptr(), kv.batch, N, Hkv, D,
        _C._code_dtype(kv.k_pool), int(block_size), P, kv.max_pages, kv.k_pool.shape[0], *strides,
        None if status is None else status.data_ptr(), dev, torch.cuda.current_stream(kv.k_pool.device).cuda_stream)
    _lib.check(rc, "build_block_meta")
    return meta


def quest_sparse_decode(Q: Tensor, kv: PagedKV, meta: Tensor, scale: float, block_size: int = 64,
                        top_k_blocks: int = 8, max_seq_len: int | None = None, return_indices: bool = False):
    """Top-k block-sparse decode with the min/max upper-bound score, exact attention inside the chosen blocks.

    Q ``[B,Hq,D]`` fp16 -> ``[B,Hq,D]`` fp16 (and the chosen block ids ``[B,Hq,top_k_blocks]`` int32).
    """
    strides = _pool_args(kv)
    _C._require(Q.is_cuda and Q.dtype == torch.float16 and Q.dim() == 3 and Q.is_contiguous(),
                "Q must be a contiguous fp16 CUDA tensor [B,Hq,D]")
    B, Hq, D = Q.shape
    _, Hkv, P, _ = kv.k_pool.shape
    _C._require(B == kv.batch, "batch mismatch between Q and the cache")
    lib = _lib.load()
    N = int(max_seq_len) if max_seq_len is not None else kv.capacity
    nb = lib.skv_quest_num_blocks(N, block_size)
    _C._require(meta.dtype == torch.float16 and meta.shape == (B, Hkv, nb, 2, D) and meta.is_contiguous(),
                "meta must be fp16 [B,Hkv,nb,2,D] built with the same block_size and max_seq_len")
    out = torch.empty((B, Hq, D), dtype=torch.float16, device=Q.device)
    idx = torch.empty((B, Hq, top_k_blocks), dtype=torch.int32, device=Q.device) if return_indices else None
    ws = _workspace.get("quest", lib.skv_quest_workspace_bytes(B, Hq, N, block_size), Q.device)
    dev = _C._dev_index(Q)
    rc = lib.skv_quest_decode(
        Q.data_ptr(), kv.k_pool.data_ptr(), kv.v_pool.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(),
        None if kv.page_table is None else kv.page_table.data_ptr(),
        None if kv.seq_lens is None else kv.seq_lens.data_ptr(), meta.data_ptr(), out.data_ptr(),
        None if idx is None else idx.data_ptr(), ws.data_ptr(), ws.numel(), B, N, Hq, Hkv, D,
        _C._code_dtype(kv.k_pool) | (_C.SKV_V_INT4 if kv.v_bits == 4 else 0), int(block_size), int(top_k_blocks), P,
        kv.max_pages, kv.k_pool.shape[0], *strides,
        float(scale), dev,
        torch.cuda.current_stream(Q.device).cuda_stream)
    _lib.check(rc, "quest_sparse_decode")
    return (out, idx) if return_indices else out


def rope_quant_append(qkv: Tensor, kv: PagedKV, Hq: int, rope_theta: float, *, meta: Tensor | None = None,
                      block_size: int = 64, status: Tensor | None = None) -> Tensor:
    """RoPE the new token's q and k, quantise k and v and store them at position ``seq_lens[b]`` of the cache.

    ``qkv`` ``[B, (Hq + 2*Hkv) * 128]`` fp16 or bf16 (fused projection output); returns the rotated query
    ``[B, Hq, 128]`` fp16.  ``kv.seq_lens`` is read, not advanced.  With ``meta`` (the tensor
    ``build_block_meta`` returns) the min/max metadata of the block that receives the token is updated in the
    same launch (``skv_rope_quant_append``).  A page-table entry outside the pool stores nothing and sets bit
    ``SKV_DEV_BAD_PAGE`` (2) in ``status`` (an int32 device tensor of one element), when one is given.  Angles are worked out
    in 32 bits (off by some 6e-8 of themselves: 0.006 radians at position 100000); :func:`append_tokens` works them out in 64.
    """
    strides = _pool_args(kv)
    _, Hkv, P, D = kv.k_pool.shape
    B = qkv.shape[0]
    _C._require(qkv.is_cuda and qkv.dim() == 2 and qkv.is_contiguous() and qkv.shape[1] == (Hq + 2 * Hkv) * D
                and qkv.dtype in (torch.float16, torch.bfloat16), "qkv must be contiguous fp16/bf16 [B,(Hq+2Hkv)*D]")
    _C._require(kv.seq_lens is not None and B == kv.batch, "the cache needs seq_lens and a matching batch")
    if meta is not None:
        _C._require(meta.dtype == torch.float16 and meta.dim() == 5 and meta.shape[:2] == (B, Hkv) and meta.shape[3:] == (2, D)
                    and meta.is_contiguous() and meta.device == qkv.device, "meta must be fp16 [B,Hkv,nb,2,D] on qkv's device")
    q = torch.empty((B, Hq, D), dtype=torch.float16, device=qkv.device)
    rc = _lib.load().skv_rope_quant_append(
        qkv.data_ptr(), int(qkv.dtype == torch.bfloat16), q.data_ptr(), kv.k_pool.data_ptr(), kv.v_pool.data_ptr(),
        kv.k_scale.data_ptr(), kv.v_scale.data_ptr(), None if kv.page_table is None else kv.page_table.data_ptr(),
        kv.seq_lens.data_ptr(), B, Hq, Hkv, D, _C._code_dtype(kv.k_pool) | (_C.SKV_V_INT4 if kv.v_bits == 4 else 0),
        P, kv.max_pages, *strides, float(rope_theta),
        None if meta is None else meta.data_ptr(), int(block_size), 0 if meta is None else meta.shape[2],
        kv.k_pool.shape[0], None if status is None else status.data_ptr(),
        _C._dev_index(qkv), torch.cuda.current_stream(qkv.device).cuda_stream)
    _lib.check(rc, "rope_quant_append")
    return q


@dataclass
class PagedKV4:
    """Paged cache whose keys and values are held in 4 bits: page records of 16 tokens, uint8 ``[num_pages, Hkv, 18, D]``
    (D 64 or 128): 9 bytes for 8 channels of a key and a value against 16.5 in the 8-bit records.

    Every 32 channels of a row share a bf16 scale ``amax / 7``.  The order of bytes inside a record is the attention
    kernel's (``skv_gqa_decode_kv4`` in the header); :func:`pack_kv4` and :func:`unpack_kv4` convert.  Fill it with
    :func:`append_tokens`.  A view of a larger buffer will do (for example one layer of ``[num_pages, layers, Hkv, 18, D]``)."""
    buf: Tensor
    page_table: Tensor | None   # int32 [B, max_pages]; None: sequence b owns pages b*max_pages ...
    seq_lens: Tensor | None     # int32 [B]
    batch: int

    page_size = 16

    @property
    def head_dim(self) -> int:
        return self.buf.shape[3]

    @property
    def max_pages(self) -> int:
        return self.page_table.shape[1] if self.page_table is not None else self.buf.shape[0] // self.batch

    @property
    def capacity(self) -> int:
        return self.max_pages * 16

    def decode(self, Q: Tensor, scale: float, *, cu_q: Tensor | None = None, max_seq_len: int | None = None,
               out: Tensor | None = None, status: Tensor | None = None) -> Tensor:
        """Dense GQA attention over the whole cache, one or several query tokens per sequence (``_C.fused_gqa_kv4``)."""
        return _C.fused_gqa_kv4(Q, self.buf, self.page_table, self.seq_lens, scale, cu_q=cu_q, max_seq_len=max_seq_len, out=out,
                                status=status)


KV4_RECORD_ROWS = 18  # rows of D bytes per (page, head): 8 of key codes, 8 of value codes, 2 of bf16 scales


def pack_kv4(k_codes: Tensor, k_scale: Tensor, v_codes: Tensor, v_scale: Tensor) -> Tensor:
    """Codes in -7..7 (int8 ``[num_pages,Hkv,16,D]``) and their bf16 scales (``[num_pages,Hkv,16,D/32]``) as page records."""
    P, H, S, D = k_codes.shape
    W = D // 32
    _C._require(S == 16 and D in (64, 128) and v_codes.shape == k_codes.shape and k_scale.shape == (P, H, 16, W)
                and v_scale.shape == k_scale.shape and k_scale.dtype == torch.bfloat16 and v_scale.dtype == torch.bfloat16,
                "4-bit page records hold [num_pages,Hkv,16,D] codes, D 64 or 128, and bf16 [num_pages,Hkv,16,D/32] scales")

    def nibbles(c):
        u = (c + 8).to(torch.uint8)
        return u[..., 0::2] | (u[..., 1::2] << 4)

    # tokens 4i + 2j + e; keys j i e c w n, values j g i e w n (see the header)
    kb = nibbles(k_codes).view(P, H, 4, 2, 2, W, 4, 4).permute(0, 1, 3, 2, 4, 6, 5, 7).reshape(P, H, 8, D)
    vb = nibbles(v_codes).view(P, H, 4, 2, 2, W, 8, 2).permute(0, 1, 3, 6, 2, 4, 5, 7).reshape(P, H, 8, D)
    sc = torch.stack([k_scale, v_scale], 3).view(P, H, 4, 2, 2, 2, W).permute(0, 1, 3, 2, 4, 5, 6).contiguous()
    return torch.cat([kb, vb, sc.view(torch.uint8).reshape(P, H, 2, D)], 2)


def unpack_kv4(buf: Tensor):
    """``(k_codes, k_scale, v_codes, v_scale)`` of page records: int8 codes and bf16 scales, the inverse of :func:`pack_kv4`."""
    P, H, R, D = buf.shape
    _C._require(R == KV4_RECORD_ROWS and D in (64, 128) and buf.dtype == torch.uint8, "not 4-bit page records")
    W = D // 32

    def codes(b):
        return (torch.stack([b & 15, b >> 4], -1).flatten(-2).to(torch.int8) - 8)

    k = codes(buf[:, :, :8].reshape(P, H, 2, 4, 2, 4, W, 4)).permute(0, 1, 3, 2, 4, 6, 5, 7).reshape(P, H, 16, D)
    v = codes(buf[:, :, 8:16].reshape(P, H, 2, 8, 4, 2, W, 2)).permute(0, 1, 4, 2, 5, 6, 3, 7).reshape(P, H, 16, D)
    sc = buf[:, :, 16:].contiguous().view(torch.bfloat16).reshape(P, H, 2, 4, 2, 2, W).permute(0, 1, 3, 2, 4, 5, 6)
    sc = sc.reshape(P, H, 16, 2, W)
    return k, sc[..., 0, :], v, sc[..., 1, :]


def _token_cache(kv):
    """Arguments of the append / read kernels that describe the cache -- the four pools, then format, page size, pages per
    sequence, pages, strides -- with the page table's pointer and (Hkv, D, device)."""
    if isinstance(kv, PagedKV4):
        b = kv.buf
        pages, Hkv, rows, D = b.shape
        sp, sh, sr, sd = b.stride()
        _C._require(b.is_cuda and b.dtype is torch.uint8 and rows == KV4_RECORD_ROWS and D in (64, 128) and sd == 1 and sr == D,
                    "not a cache of 4-bit page records")
        pools, layout, dev = (b.data_ptr(), None, None, None), (_lib.KV_INT4, 16, kv.max_pages, pages, sp, sh, 0, 0, 0), b.device
    else:
        strides = _pool_args(kv)
        pages, Hkv, size, D = kv.k_pool.shape
        pools = (kv.k_pool.data_ptr(), kv.v_pool.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr())
        layout = (_C._code_dtype(kv.k_pool) | (_C.SKV_V_INT4 if kv.v_bits == 4 else 0), size, kv.max_pages, pages, *strides)
        dev = kv.k_pool.device
    table = kv.page_table
    if table is not None:
        _C._require(table.dtype is torch.int32 and table.dim() == 2 and table.shape[0] == kv.batch and table.is_contiguous()
                    and table.device == dev, "page_table must be a contiguous int32 [B,max_pages] tensor on the cache's device")
        table = table.data_ptr()
    else:
        _C._require(pages % kv.batch == 0, "without a page table num_pages must be B * max_pages")
    return pools, layout, table, Hkv, D, dev


def _int32(t: Tensor, n: int, dev, what: str) -> int:
    """Pointer of an int32 argument.  The caller keeps the tensor under its own name until the launch: one made in the call would
    else be freed here, and its memory given to the outputs that are allocated next."""
    if not (t.dtype is torch.int32 and t.shape == (n,) and t.is_contiguous() and t.device == dev):
        raise RuntimeError(f"{what} must be a contiguous int32 [{n}] tensor on the cache's device")
    return t.data_ptr()


def append_tokens(qkv: Tensor, kv: "PagedKV | PagedKV4", Hq: int, rope=None, *, cu_new: Tensor | None = None,
                  positions: Tensor | None = None, q_out: Tensor | None = None, status: Tensor | None = None) -> Tensor:
    """Rotate, quantise and store any number of new tokens per sequence: a prompt, a chunk of one, drafted tokens, a step.

    ``qkv`` ``[T, (Hq + 2*Hkv) * D]`` fp16 or bf16 (fused projection output; rows may be strided).  Rows
    ``cu_new[b]..cu_new[b+1]`` (int32 ``[B+1]``; ``None``: one row per sequence) are the next tokens of sequence b and take
    positions ``kv.seq_lens[b]``, ``+ 1``, ...; ``seq_lens`` is read, not advanced.  ``rope`` (a ``RotaryEmbedding``;
    ``None``: no rotation) turns q and k at those positions, or at ``positions`` (int32 or int64 ``[T]``) where the place in
    the cache is not the place in the text (an evicted, compacted cache).  Returns the rotated query ``[T, Hq, D]``: fp16, or
    ``q_out`` (fp16 or bf16).  Rows before ``cu_new[0]`` and from ``cu_new[B]`` on belong to no sequence (part of a batch, padding)
    and are left alone.  Tokens past a sequence's page list are not stored;
    neither is one whose page-table entry lies outside the pool, which sets ``SKV_DEV_BAD_PAGE`` (2) in ``status`` (an
    int32 device tensor of one element).  Serves ``PagedKV4`` (D 64 or 128) and every ``PagedKV`` (D 128); a rotary width
    must be a multiple of 16 (interleaved: of 8).  Block metadata is not kept current: rebuild it (``build_block_meta``).
    Scales are ``amax * fp32(1 / top code)`` in every format, as torch divides by a number on the GPU; ``rope_quant_append`` divides
    and has 32-bit angles, so the two may differ in a scale's last bit and, at far positions, in the angle: fill a sequence by
    one of them.
    """
    pools, layout, table, Hkv, D, dev = _token_cache(kv)
    bf16 = qkv.dtype is torch.bfloat16
    _C._require(qkv.device == dev and qkv.dim() == 2 and (bf16 or qkv.dtype is torch.float16) and Hq >= 0
                and qkv.shape[1] == (Hq + 2 * Hkv) * D and qkv.stride(1) == 1,
                "qkv must be fp16/bf16 [T,(Hq+2Hkv)*D] on the cache's device, channels contiguous")
    T, B = qkv.shape[0], kv.batch
    _C._require(kv.seq_lens is not None, "the cache needs seq_lens")
    lens = _int32(kv.seq_lens, B, dev, "seq_lens")
    cu = pos = None
    if cu_new is None:
        _C._require(T == B, "one row per sequence, or cu_new")
    else:
        cu = _int32(cu_new, B + 1, dev, "cu_new")
    freqs, width, inter, factor = (None, 0, 0, 1.0) if rope is None else rope.kernel_args(D, dev)
    pos64 = False
    if positions is not None:
        pos64 = positions.dtype is torch.int64
        _C._require((pos64 or positions.dtype is torch.int32) and positions.shape == (T,) and positions.is_contiguous()
                    and positions.device == dev, "positions must be a contiguous int32 or int64 [T] tensor on the cache's device")
        pos = positions.data_ptr()
    if q_out is None:
        q_out, q_bf16 = qkv.new_empty((T, Hq, D), dtype=torch.float16), False
    else:
        q_bf16 = q_out.dtype is torch.bfloat16
        _C._require((q_bf16 or q_out.dtype is torch.float16) and q_out.shape == (T, Hq, D) and q_out.is_contiguous()
                    and q_out.device == dev, "q_out must be a contiguous fp16 or bf16 [T,Hq,D] tensor on the cache's device")
    rc = _lib.load().skv_append_tokens(
        qkv.data_ptr(), bf16, qkv.stride(0) if T > 1 else qkv.shape[1], q_out.data_ptr(), q_bf16, freqs, width, inter, factor,
        pos, pos64, cu, table, lens, *pools, T, B, Hq, Hkv, D, *layout,
        None if status is None else _int32(status, 1, dev, "status"), dev.index, _workspace.stream(dev.index))
    if rc:
        _lib.check(rc, "append_tokens")
    return q_out


def read_tokens(kv: "PagedKV | PagedKV4", cu: Tensor, rows: int, *, starts: Tensor | None = None,
                dtype: torch.dtype = torch.float16, status: Tensor | None = None):
    """Rows of cached tokens as values: ``(K, V)`` ``[rows, Hkv, D]`` fp16 or bf16, code times scale rounded once.

    Rows ``cu[b]..cu[b+1]`` (int32 ``[B+1]``, ``cu[B] <= rows``) are positions ``starts[b]``, ``+ 1``, ... (int32 ``[B]``;
    ``None``: from 0) of sequence b: the prefix that a chunk of prompt attends to through another kernel, or a check of what
    was stored.  ``kv.seq_lens`` is not consulted.  Rows before ``cu[0]`` and from ``cu[B]`` on are not written; a position without a page reads as
    zeros (``status`` as in :func:`append_tokens`)."""
    pools, layout, table, Hkv, D, dev = _token_cache(kv)
    _C._require((dtype is torch.float16 or dtype is torch.bfloat16) and rows >= 0, "read_tokens returns fp16 or bf16 rows")
    B = kv.batch
    offsets = _int32(cu, B + 1, dev, "cu")
    K = torch.empty((rows, Hkv, D), dtype=dtype, device=dev)
    V = torch.empty_like(K)
    rc = _lib.load().skv_read_tokens(
        *pools, table, offsets, None if starts is None else _int32(starts, B, dev, "starts"), K.data_ptr(), V.data_ptr(),
        dtype is torch.bfloat16, rows, B, Hkv, D, *layout, None if status is None else _int32(status, 1, dev, "status"),
        dev.index, _workspace.stream(dev.index))
    if rc:
        _lib.check(rc, "read_tokens")
    return K, V


def repage_evicted(res, *, pool: Tensor | None = None, page_ids: Tensor | None = None) -> PagedKV:
    """Put the compacted, quantised output of ``fused_kv_evict`` back into paged form (page reclamation).

    ``res`` is the ``EvictionResult`` of a scaled-quantisation eviction in position order: codes
    ``[B, H, keep, 128]`` (int8 or e4m3) and fp32 scales ``[B, H, keep]``.  Slot ``j`` of every head's new
    sequence is that head's ``j``-th kept token (heads keep different positions; the keys already carry their
    rotary phase, so attention does not need the original positions).  The rows are written as fused page
    records of 16 tokens, either into fresh storage or -- with ``pool`` (a fused page-record buffer) and
    ``page_ids`` (int ``[B, ceil(keep/16)]``, the pages handed out by the caller's allocator) -- into an
    existing pool; the pages the sequences occupied before are then free for reuse.  Returns the ``PagedKV``
    with ``seq_lens = keep``.
    """
    K, V, ks, vs = res.K, res.V, res.k_scale, res.v_scale
    _C._require(ks is not None and vs is not None, "repage_evicted needs a scaled (int8 or fp8) eviction result")
    B, H, keep, D = K.shape
    _C._require(D == 128, "page records hold 128-channel rows")
    n = (keep + 15) // 16
    pad = n * 16 - keep

    def rows(t):      # [B,H,keep,...] -> [B*n, H, 16, ...]
        if pad:
            t = torch.cat([t, t.new_zeros((B, H, pad) + tuple(t.shape[3:]))], dim=2)
        t = t.reshape((B, H, n, 16) + tuple(t.shape[3:]))
        return t.permute(0, 2, 1, 3, *range(4, t.dim())).reshape((B * n, H, 16) + tuple(t.shape[4:]))

    code_dtype = K.dtype
    records = pack_fused(rows(K.view(torch.uint8)).view(code_dtype), rows(V.view(torch.uint8)).view(code_dtype),
                         rows(ks), rows(vs))
    if pool is None:
        table = torch.arange(B * n, dtype=torch.int32, device=K.device).view(B, n)
        buf = records
    else:
        _C._require(page_ids is not None and tuple(page_ids.shape) == (B, n), "page_ids must be [B, ceil(keep/16)]")
        _C._require(pool.dtype == torch.uint8 and pool.dim() == 4 and tuple(pool.shape[1:]) == (H, RECORD_ROWS, 128),
                    "pool must be a fused page-record buffer [num_pages, H, 33, 128]")
        pool[page_ids.reshape(-1).long()] = records
        table = page_ids.to(torch.int32).contiguous()
        buf = pool
    lens = torch.full((B,), keep, dtype=torch.int32, device=K.device)
    return PagedKV.from_fused(buf, code_dtype, table, lens, B)
