"""Paged K/V cache of the text layers: the pool of pages and the sequences of
a batch, as the handles that `ops.cache_write`, `ops.cache_read` and
`ops.cache_attention` take.

piR2 prefills one observation per robot and keeps no K/V cache (its VLM runs
transformers' "sdpa" attention without one, coexecution/optimization/groot/
vlm.py:312-313).  These serve several robots whose prompts differ in length
and grow afterwards: each sequence owns pages of a shared pool, in bf16, or
as int8 / E4M3 codes with one fp32 scale per token and head (the arithmetic
of the symmetric-row-v1 activation pack), or in 4 bits: codes of -7..7, an E4M3
factor for every 32 channels and one power of two per token and head.
"""

import ctypes

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
FORMATS = {
    torch.bfloat16: _lib.CACHE_BF16, torch.int8: _lib.CACHE_INT8, torch.float8_e4m3fn: _lib.CACHE_E4M3,
    torch.uint8: _lib.CACHE_INT4,
}
FACTOR_GROUP = 32   # channels of a 4-bit row that share a factor


def rotary_table(positions, head_dim, theta=1e4, *, device="cuda"):
    """(cos, sin) fp32 [positions, head_dim / 2] of the angles p theta^(-2 i /
    head_dim), as `ops.cache_append` takes them; the angles are computed in 64
    bits (in 32, those of far positions are off by 2^-24 of many turns)."""
    if positions < 1 or head_dim not in HEAD_DIMS:
        raise ValueError(f"rotary_table: positions must be at least 1, head_dim one of {HEAD_DIMS}")
    inverse = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
    angles = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), inverse)
    return angles.cos().float(), angles.sin().float()


class KVPages:
    """One layer's pool: k, v [pages, kv_heads, page_size, head_dim] of one
    dtype (bfloat16, int8 or float8_e4m3fn; uint8 [..., head_dim / 2] holds 4-bit
    codes, the even channel in the low bits) and, for the quantised ones, fp32
    scales [pages, kv_heads, page_size]; 4-bit pages also have factors,
    float8_e4m3fn [pages, kv_heads, page_size, head_dim / 32].  Pages may lie
    apart (any stride of the first dimension, so that all layers share one
    allocation); inside a page everything is contiguous."""

    def __init__(self, k, v, k_scale=None, v_scale=None, k_factor=None, v_factor=None):
        if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in FORMATS:
            raise ValueError("KVPages: k and v must be [pages, kv_heads, page_size, head_dim] bf16, int8 or float8_e4m3fn, or uint8 of 4-bit codes")
        pages, heads, size, wide = k.shape
        packed = k.dtype == torch.uint8
        dim = 2 * wide if packed else wide
        if pages < 1 or heads < 1 or size not in PAGE_SIZES or dim not in HEAD_DIMS:
            raise ValueError(f"KVPages: page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
        quantised = k.dtype != torch.bfloat16
        if quantised != (k_scale is not None) or quantised != (v_scale is not None):
            raise ValueError("KVPages: 8-bit and 4-bit pages need k_scale and v_scale, bf16 pages take none")
        if packed != (k_factor is not None) or packed != (v_factor is not None):
            raise ValueError("KVPages: 4-bit pages need k_factor and v_factor, others take none")
        tensors = [k, v] + ([k_scale, v_scale] if quantised else []) + ([k_factor, v_factor] if packed else [])
        if any(not t.is_cuda or t.device != k.device for t in tensors):
            raise ValueError("KVPages: all tensors must be on one CUDA device")
        for t in (k, v):
            if t.stride()[1:] != (size * wide, wide, 1) or (pages > 1 and t.stride(0) < heads * size * wide):
                raise ValueError("KVPages: pages must be contiguous and apart")
        for t in tensors[2:4]:
            if t.shape != (pages, heads, size) or t.dtype != torch.float32:
                raise ValueError("KVPages: scales must be fp32 [pages, kv_heads, page_size]")
            if t.stride()[1:] != (size, 1) or (pages > 1 and t.stride(0) < heads * size):
                raise ValueError("KVPages: scales of a page must be contiguous and apart")
        groups = dim // FACTOR_GROUP
        for t in tensors[4:]:
            if t.shape != (pages, heads, size, groups) or t.dtype != torch.float8_e4m3fn:
                raise ValueError("KVPages: factors must be float8_e4m3fn [pages, kv_heads, page_size, head_dim / 32]")
            if t.stride()[1:] != (size * groups, groups, 1) or (pages > 1 and t.stride(0) < heads * size * groups):
                raise ValueError("KVPages: factors of a page must be contiguous and apart")

        def apart(t, size_of_page):
            return t.stride(0) if pages > 1 else size_of_page

        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.k_factor, self.v_factor = k_factor, v_factor
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self.dtype, self.device, self.index = k.dtype, k.device, k.get_device()
        self.struct = _lib.KVPagesStruct(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if quantised else None,
            v_scale.data_ptr() if quantised else None, apart(k, heads * size * wide), apart(v, heads * size * wide),
            apart(k_scale, heads * size) if quantised else 0, apart(v_scale, heads * size) if quantised else 0,
            pages, size, heads, dim, FORMATS[k.dtype],
            k_factor.data_ptr() if packed else None, v_factor.data_ptr() if packed else None,
            apart(k_factor, heads * size * groups) if packed else 0, apart(v_factor, heads * size * groups) if packed else 0,
        )
        self.address = ctypes.addressof(self.struct)
        self.blank = torch.empty(0, dtype=torch.bfloat16, device=k.device)   # what reads allocate like

    @classmethod
    def allocate(cls, pages, kv_heads, head_dim, *, page_size=64, dtype=torch.int8, device="cuda"):
        """A pool of its own allocation, zeroed; dtype uint8: of 4-bit codes."""
        packed = dtype == torch.uint8
        shape = (pages, kv_heads, page_size, head_dim // 2 if packed else head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype == torch.bfloat16:
            return cls(k, v)
        scales = [torch.ones(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        groups = (*shape[:3], head_dim // FACTOR_GROUP)
        factors = [torch.zeros(groups, dtype=torch.float8_e4m3fn, device=device) for _ in range(2 if packed else 0)]
        return cls(k, v, *scales, *factors)


class Sequences:
    """The sequences of a batch: `starts` int32 [batch + 1], the packed rows
    of each; `lengths` int32 [batch], the tokens it has in the cache once
    those rows are in it; `table` int32 [batch, width], the page of each
    page_size positions (entries past a sequence's length are not read).  The
    tensors may be rewritten in place between calls (and between replays of a
    captured graph); the kernels check every index against table and pool."""

    def __init__(self, starts, lengths, table):
        for t, ndim in ((starts, 1), (lengths, 1), (table, 2)):
            if not t.is_cuda or t.dtype != torch.int32 or t.ndim != ndim or t.device != starts.device:
                raise ValueError("Sequences: starts [batch + 1], lengths [batch] and table [batch, width] must be int32 on one CUDA device")
        batch, width = table.shape
        if batch < 1 or width < 1 or lengths.shape != (batch,) or starts.shape != (batch + 1,):
            raise ValueError("Sequences: starts must have batch + 1 entries, lengths and table batch rows, table a column")
        if not starts.is_contiguous() or not lengths.is_contiguous() or table.stride(1) != 1 or (batch > 1 and table.stride(0) < width):
            raise ValueError("Sequences: starts and lengths must be contiguous, table have contiguous rows")
        self.starts, self.lengths, self.table = starts, lengths, table
        self.batch, self.width = batch, width
        self.device, self.index = starts.device, starts.get_device()
        self.struct = _lib.SequencesStruct(
            starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), table.stride(0) if batch > 1 else width, batch, width
        )
        self.address = ctypes.addressof(self.struct)
