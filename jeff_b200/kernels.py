"""The hot path's operators as the reference's fast path calls them, each one call into libjeffb200 (no Triton, no
CPU fallback). Names, arguments and returns follow the reference's engine modules:

- int4_product (int4_kernels.py:132-177), lora_shrink (fast_path.py:159-177): the fused W4A16 + multi-LoRA product;
- add_rms, gated_norm, gate_mul, silu_mul (fast_path.py:80-156), rms_last (batched_path.py:274-275), embed;
- gdn_prep_rows, gdn_scan (batched_kernels.py:89-261 and fla's chunk kernel), attn_prep_rows, paged_attention,
  kv_scatter (batched_kernels.py:302-486, batched_path.py:345-349), readout_rows (batched_kernels.py:492-559);
- block_tables, attn_prep_axes, decode_attention, linear_scan, linear_step: single tokens over the prefix pool and
  linear attention with a decay for each head, which the reference does not have. They take the pool's typed views
  (PrefixPool.kv, PrefixPool.state), whose strides say where a page lies, and run on their tensors' device.

Every function launches on the current torch stream and allocates its outputs only when no `out` is given (the
recorded passes pass preallocated buffers, so graphs capture no allocation)."""

from __future__ import annotations

import functools
from collections.abc import Sequence
from typing import NamedTuple

import torch

from jeff_b200 import _lib
from jeff_b200 import constants as C
from jeff_b200._lib import ptr, stream_ptr

DT = torch.bfloat16


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...] | None = None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor, got strides {t.stride()}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")


def _pass_rows(t: int, n: int) -> int:
    if n % 32 or t % n:
        raise ValueError(f"A pass of {t} tokens in rows of {n}: rows must be a multiple of 32 tokens, and the pass "
                         "whole rows")
    return t // n


# ---------------------------------------------------------------- int4 products


def int4_repack(words: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The reference's kernel word layout -> this library's kernel layout (jb_int4_repack), on the device."""
    out = out if out is not None else torch.empty_like(words)
    _lib.call("jb_int4_repack", ptr(words), ptr(out), words.shape[0] * 8, words.shape[1], stream_ptr())
    return out


def int4_dequant(words: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int) -> torch.Tensor:
    """The packed group (kernel-layout words) dequantised on the device: (columns, k) bf16."""
    k, columns = words.shape[0] * 8, words.shape[1]
    out = torch.empty(columns, k, dtype=DT, device=words.device)
    _lib.call("jb_int4_dequant", ptr(words), ptr(scales), ptr(zeros), k, columns, group, ptr(out), stream_ptr())
    return out


def lora_shrink(x: torch.Tensor, lora_a: torch.Tensor, adapters: torch.Tensor, row_len: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    m, k = x.shape
    rank = lora_a.shape[1]
    mid = out if out is not None else torch.empty(m, rank, dtype=DT, device=x.device)
    _lib.call("jb_lora_shrink", ptr(x), m, k, ptr(lora_a), rank, lora_a.shape[0], ptr(adapters), row_len, ptr(mid),
              stream_ptr())
    return mid


def int4_product(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int,
                 out_features: int, lora_a: torch.Tensor | None, lora_b: torch.Tensor | None,
                 adapters: torch.Tensor | None, row_len: int, mid: torch.Tensor | None = None,
                 y: torch.Tensor | None = None, swiglu: bool = False, tmem_a: bool = False,
                 split: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """y (m, out) = bf16(x W^T + bf16(x A[a]^T) B[a]^T) for row a = adapters[t // row_len] of token t: the fused
    product of one group (module docstring); `words` in the kernel layout (int4_repack). lora_a (rows, R, k),
    lora_b (rows, columns, R) bf16, or None. swiglu: the group's columns are gate|up blocks of 64 and y (m, out / 2)
    receives bf16(bf16(silu(g)) u) (fast_path.silu_mul fused into the epilogue). tmem_a: the tensor-memory form of
    the product kernel (weights dequantised into tensor memory as the MMA's A operand; the same bits, measured
    slower), for rows of a multiple of 128 tokens. split (fp32 slices, int32 counters, the counters zero): the
    split-K form (jb_int4_lora_product_split), which the library uses when the pass's tiles are fewer than the SMs;
    the same result up to the order of the fp32 sums."""
    m, k = x.shape
    columns = words.shape[1]
    if words.shape[0] * 8 != k:
        raise ValueError(f"int4_product: x has {k} inputs, the weights {words.shape[0] * 8}")
    rank = 0 if lora_a is None else lora_a.shape[1]
    if y is None:
        y = torch.empty(m, out_features // 2 if swiglu else out_features, dtype=DT, device=x.device)
    if rank and mid is None:
        mid = torch.empty(m, rank, dtype=DT, device=x.device)
    args = (ptr(x), m, k, ptr(words), ptr(scales), ptr(zeros), group, columns, out_features, ptr(lora_a), ptr(lora_b),
            rank, 0 if lora_a is None else lora_a.shape[0], ptr(adapters), row_len, ptr(mid) if rank else None, ptr(y),
            y.stride(0), (1 if swiglu else 0) | (2 if tmem_a else 0))
    if split is None:
        _lib.call("jb_int4_lora_product", *args, stream_ptr())
    else:
        parts, counters = split
        _check(parts, "split partials", torch.float32)
        _check(counters, "split counters", torch.int32)
        _lib.call("jb_int4_lora_product_split", *args, ptr(parts), parts.numel(), ptr(counters), counters.numel(),
                  stream_ptr())
    return y


def w4a16_small(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int,
                out_features: int, mid: torch.Tensor | None, lora_b: torch.Tensor | None,
                adapters: torch.Tensor | None, row_len: int, split: int = 0, swiglu: bool = False,
                y: torch.Tensor | None = None) -> torch.Tensor:
    """The weight-streaming product for passes of at most 64 tokens in at most two LoRA rows (jb_w4a16_lora_small):
    y = bf16(x W^T + mid B[a]^T), mid the LoRA first factor (m, R) already computed (or None). split: K slices per
    128-column tile, one thread-block cluster (0: the library's choice)."""
    m, k = x.shape
    columns = words.shape[1]
    rank = 0 if mid is None else mid.shape[1]
    if y is None:
        y = torch.empty(m, out_features // 2 if swiglu else out_features, dtype=DT, device=x.device)
    _lib.call("jb_w4a16_lora_small", ptr(x), m, k, ptr(words), ptr(scales), ptr(zeros), group, columns, out_features,
              ptr(mid), ptr(lora_b), rank, 0 if lora_b is None else lora_b.shape[0], ptr(adapters), row_len, ptr(y),
              y.stride(0), 1 if swiglu else 0, split, stream_ptr())
    return y


# ---------------------------------------------------------------- norms and activations


def add_rms(x: torch.Tensor, d: torch.Tensor | None, w1: torch.Tensor, xo: torch.Tensor | None = None,
            h: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(x + d, rms(x + d) * w1), w1 = 1 + weight float32 (fast_path.add_rms)."""
    rows, n = x.shape
    h = h if h is not None else torch.empty_like(x)
    if d is not None:
        xo = xo if xo is not None else torch.empty_like(x)
    else:
        xo = x
    _lib.call("jb_add_rms", ptr(x), ptr(d), ptr(w1), ptr(xo), ptr(h), rows, n, stream_ptr())
    return xo, h


def rms_last(x: torch.Tensor, d: torch.Tensor, last: torch.Tensor, row_len: int, w1: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
    b = x.shape[0] // row_len
    hidden = out if out is not None else torch.empty(b, x.shape[1], dtype=DT, device=x.device)
    _lib.call("jb_rms_last", ptr(x), ptr(d), ptr(last), b, row_len, x.shape[1], ptr(w1), ptr(hidden), stream_ptr())
    return hidden


def embed(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    t = ids.shape[0]
    x = out if out is not None else torch.empty(t, table.shape[1], dtype=DT, device=table.device)
    _lib.call("jb_embed", ptr(table), table.shape[0], table.shape[1], ptr(ids), t, ptr(x), stream_ptr())
    return x


def silu_mul(gu: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    rows = gu.shape[0]
    y = out if out is not None else torch.empty(rows, C.INTER, dtype=DT, device=gu.device)
    _lib.call("jb_silu_mul", ptr(gu), gu.stride(0), C.INTER, ptr(y), rows, stream_ptr())
    return y


def gate_mul(o: torch.Tensor, pr: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    rows = pr.shape[0]
    y = out if out is not None else torch.empty(rows, C.NQ * C.HD, dtype=DT, device=o.device)
    _lib.call("jb_gate_mul", ptr(o), ptr(pr), pr.stride(0), ptr(y), rows, stream_ptr())
    return y


def gated_norm(o: torch.Tensor, pr: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    rows = pr.shape[0]
    y = out if out is not None else torch.empty(rows, C.NV * C.DV, dtype=DT, device=o.device)
    _lib.call("jb_gated_norm", ptr(o), ptr(pr), pr.stride(0), C.QKV_DIM, ptr(w), ptr(y), rows, stream_ptr())
    return y


def readout_rows(hidden: torch.Tensor, readout_pool: torch.Tensor, temp_pool: torch.Tensor, adapters: torch.Tensor,
                 counts: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Each row's option probabilities (B, 255) fp32 (batched_kernels.readout_rows)."""
    b = hidden.shape[0]
    if temp_pool.dim() != 1 or temp_pool.dtype != torch.float32 or not temp_pool.is_contiguous():
        raise ValueError(f"readout_rows: temp_pool must be a contiguous float32 vector (one temperature per adapter "
                         f"row), got shape {tuple(temp_pool.shape)}, {temp_pool.dtype}")
    if readout_pool.shape[1:] != (C.READOUT_ROWS, C.HIDDEN) or not readout_pool.is_contiguous():
        raise ValueError(f"readout_rows: expected a contiguous readout_pool (adapters + 1, {C.READOUT_ROWS}, "
                         f"{C.HIDDEN}), got {tuple(readout_pool.shape)}")
    probs = out if out is not None else torch.empty(b, C.READOUT_ROWS, dtype=torch.float32, device=hidden.device)
    _lib.call("jb_readout_rows", ptr(hidden), ptr(readout_pool), readout_pool.shape[0], ptr(temp_pool), ptr(adapters),
              ptr(counts), b, ptr(probs), stream_ptr())
    return probs


# ---------------------------------------------------------------- Gated DeltaNet


def gdn_prep_rows(pr: torch.Tensor, pool, tables: torch.Tensor, gdn_layer: int, conv_w: torch.Tensor,
                  a_neg: torch.Tensor, dt_bias: torch.Tensor, n: int, real: torch.Tensor | None = None,
                  out_tables: torch.Tensor | None = None, outs: tuple | None = None) -> tuple[torch.Tensor, ...]:
    """q, k, v (B, n, 16, 128) bf16, g (B, n, 16) fp32, beta (B, n, 16) bf16 (batched_kernels.gdn_prep_rows).
    With real and out_tables (the prefix pass): padding tokens get g = beta = 0 and each row's conv tail goes to its
    output pages."""
    t = pr.shape[0]
    b = _pass_rows(t, n)
    shapes = pool.shapes
    if tables.dim() != 2 or tables.shape[0] < b or tables.shape[1] < shapes.fixed_pages or tables.dtype != torch.int32:
        raise ValueError(f"tables: expected int32 (rows >= {b}, width >= {shapes.fixed_pages}), got "
                         f"{tuple(tables.shape)} {tables.dtype}")
    if conv_w.shape != (4, C.QKV_DIM) or conv_w.dtype != torch.float32 or not conv_w.is_contiguous():
        raise ValueError(f"gdn_prep_rows: conv_w must be a contiguous float32 (4, {C.QKV_DIM}) tensor, got "
                         f"{tuple(conv_w.shape)}, {conv_w.dtype}")
    for name, vec in (("a", a_neg), ("dt_bias", dt_bias)):
        if vec.shape != (C.NV,) or vec.dtype != torch.float32 or not vec.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous torch.float32 vector of {C.NV} entries, got shape "
                             f"{tuple(vec.shape)}, {vec.dtype}")
    dev = pr.device
    if outs is None:
        q = torch.empty(b, n, C.NV, C.DK, dtype=DT, device=dev)
        outs = (q, torch.empty_like(q), torch.empty_like(q), torch.empty(b, n, C.NV, dtype=torch.float32, device=dev),
                torch.empty(b, n, C.NV, dtype=DT, device=dev))
    q, k, v, g, beta = outs
    per = shapes.layers_per_conv_page
    _lib.call("jb_gdn_prep_rows", ptr(pr), pr.stride(0), t, n, ptr(pool.data), shapes.page_bytes, ptr(tables),
              tables.stride(0), shapes.state_pages + gdn_layer // per, gdn_layer % per, ptr(conv_w), ptr(a_neg),
              ptr(dt_bias), ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(real), ptr(out_tables),
              0 if out_tables is None else out_tables.stride(0), stream_ptr())
    return q, k, v, g, beta


def gdn_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, pool,
             tables: torch.Tensor, gdn_layer: int, last: torch.Tensor | None = None,
             out_tables: torch.Tensor | None = None, out: torch.Tensor | None = None,
             kernel: str = "tc") -> torch.Tensor:
    """The gated delta rule from each row's pooled state; o (B, n, 16, 128). kernel "tc" (64-token chunks, every
    chunk product a tcgen05 MMA with the state in tensor memory: fla's chunk_gated_delta_rule), "chunk" (the same
    chunks on mma.sync, the form the fused jb_gdn_layer shares bit for bit) or "recurrent" (token by token,
    batched_kernels.gdn_recurrent_slots)."""
    b, n = q.shape[:2]
    shapes = pool.shapes
    if tables.dim() != 2 or tables.shape[0] < b or tables.shape[1] < shapes.fixed_pages or tables.dtype != torch.int32:
        raise ValueError(f"tables: expected int32 (rows >= {b}, width >= {shapes.fixed_pages}), got "
                         f"{tuple(tables.shape)} {tables.dtype}")
    for name, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        if not x.is_contiguous():
            raise ValueError(f"gdn_scan: {name} must be contiguous")
    o = out if out is not None else torch.empty_like(v)
    name = {"tc": "jb_gdn_scan_tc", "chunk": "jb_gdn_scan", "recurrent": "jb_gdn_scan_recurrent"}[kernel]
    _lib.call(name, ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(o), b, n, ptr(pool.data),
              shapes.page_bytes, ptr(tables), tables.stride(0), shapes.state[0] * gdn_layer, shapes.heads_per_page,
              ptr(last), ptr(out_tables), 0 if out_tables is None else out_tables.stride(0), stream_ptr())
    return o


def gdn_layer(pr: torch.Tensor, pool, tables: torch.Tensor, gdn_layer: int, conv_w: torch.Tensor,
              a_neg: torch.Tensor, dt_bias: torch.Tensor, gnorm_w: torch.Tensor, n: int,
              last: torch.Tensor | None = None, real: torch.Tensor | None = None,
              out_tables: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A Gated DeltaNet layer's mixer in one launch (gdn_prep_rows, the chunked rule and gated_norm fused): y
    (t, 2048) bf16 from the in_proj output pr (t, 8224), each row resuming from its pooled state and conv tail.
    last: the decision pass's last real token per row; real + out_tables: the prefix pass."""
    t = pr.shape[0]
    _pass_rows(t, n)
    shapes = pool.shapes
    if tables.dim() != 2 or tables.shape[0] < t // n or tables.shape[1] < shapes.fixed_pages or \
            tables.dtype != torch.int32:
        raise ValueError(f"tables: expected int32 (rows >= {t // n}, width >= {shapes.fixed_pages}), got "
                         f"{tuple(tables.shape)} {tables.dtype}")
    if conv_w.shape != (4, C.QKV_DIM) or conv_w.dtype != torch.float32 or not conv_w.is_contiguous():
        raise ValueError(f"gdn_layer: conv_w must be a contiguous float32 (4, {C.QKV_DIM}) tensor, got "
                         f"{tuple(conv_w.shape)}, {conv_w.dtype}")
    if gnorm_w.shape != (C.DV,) or gnorm_w.dtype != DT or not gnorm_w.is_contiguous():
        raise ValueError(f"gdn_layer: gnorm_w must be a contiguous bf16 ({C.DV},) vector")
    if pr.stride(1) != 1 or pr.shape[1] < C.GDN_PROJ:
        raise ValueError(f"gdn_layer: pr must be row-major with at least {C.GDN_PROJ} columns")
    y = out if out is not None else torch.empty(t, C.NV * C.DV, dtype=DT, device=pr.device)
    if y.stride(1) != 1 or y.shape[1] < C.NV * C.DV:
        raise ValueError("gdn_layer: out must be row-major with at least 2048 columns")
    per = shapes.layers_per_conv_page
    _lib.call("jb_gdn_layer", ptr(pr), pr.stride(0), t, n, ptr(pool.data), shapes.page_bytes, ptr(tables),
              tables.stride(0), shapes.state[0] * gdn_layer, shapes.heads_per_page, shapes.state_pages + gdn_layer // per,
              gdn_layer % per, ptr(conv_w), ptr(a_neg), ptr(dt_bias), ptr(gnorm_w), ptr(y), y.stride(0), ptr(last),
              ptr(real), ptr(out_tables), 0 if out_tables is None else out_tables.stride(0), stream_ptr())
    return y


# ---------------------------------------------------------------- attention


def attn_prep_rows(pr: torch.Tensor, q_w1: torch.Tensor, k_w1: torch.Tensor, inv_freq: torch.Tensor,
                   pos: torch.Tensor, kn: torch.Tensor, vn: torch.Tensor, n: int,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    t = pr.shape[0]
    _pass_rows(t, n)
    for name, x in (("kn", kn), ("vn", vn)):
        if tuple(x.shape) != (t, C.NKV, C.HD) or not x.is_contiguous():
            raise ValueError(f"attn_prep_rows: {name} must be a contiguous ({t}, {C.NKV}, {C.HD}) tensor")
    q = out if out is not None else torch.empty(t, C.NQ, C.HD, dtype=DT, device=pr.device)
    _lib.call("jb_attn_prep_rows", ptr(pr), pr.stride(0), t, n, ptr(q_w1), ptr(k_w1), ptr(inv_freq), ptr(pos), ptr(q),
              ptr(kn), ptr(vn), stream_ptr())
    return q


def paged_attention(q: torch.Tensor, pool, tables: torch.Tensor, attn_layer: int, pos: torch.Tensor,
                    kn: torch.Tensor, vn: torch.Tensor, n: int, out: torch.Tensor | None = None) -> torch.Tensor:
    t = q.shape[0]
    b = _pass_rows(t, n)
    width = pool.fixed_pages + pool.max_kv_pages
    if tables.dim() != 2 or tables.shape[0] < b or tables.shape[1] < width or tables.dtype != torch.int32:
        raise ValueError(f"tables: expected int32 (rows >= {b}, width >= {width}), got {tuple(tables.shape)} "
                         f"{tables.dtype}")
    for name, x in (("q", q), ("kn", kn), ("vn", vn)):
        if not x.is_contiguous():
            raise ValueError(f"paged_attention: {name} must be contiguous")
    o = out if out is not None else torch.empty(t, C.NQ, C.HD, dtype=DT, device=q.device)
    _lib.call("jb_paged_attention", ptr(q), ptr(pool.data), pool.shapes.page_bytes, ptr(tables), tables.stride(0),
              pool.fixed_pages, attn_layer, pool.shapes.attn_layers, ptr(pos), ptr(kn), ptr(vn), ptr(o), b, n,
              stream_ptr())
    return o


def paged_attention_gated(q: torch.Tensor, pool, tables: torch.Tensor, attn_layer: int, pos: torch.Tensor,
                          kn: torch.Tensor, vn: torch.Tensor, n: int, pr: torch.Tensor,
                          out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Paged prefix-KV attention on tcgen05 with the output gate fused (paged_attention then gate_mul in one launch):
    y (t, 2048) bf16 = bf16(bf16(attention) * bf16(sigmoid(gate))), the gate half of each head's q_proj output in
    pr. scratch (fp32): the split walk's (jb_paged_attention_gated_split), which passes too small to fill the GPU
    spread over more CTAs."""
    t = q.shape[0]
    b = _pass_rows(t, n)
    width = pool.fixed_pages + pool.max_kv_pages
    if tables.dim() != 2 or tables.shape[0] < b or tables.shape[1] < width or tables.dtype != torch.int32:
        raise ValueError(f"tables: expected int32 (rows >= {b}, width >= {width}), got {tuple(tables.shape)} "
                         f"{tables.dtype}")
    for name, x in (("q", q), ("kn", kn), ("vn", vn)):
        if not x.is_contiguous():
            raise ValueError(f"paged_attention_gated: {name} must be contiguous")
    y = out if out is not None else torch.empty(t, C.NQ * C.HD, dtype=DT, device=q.device)
    args = (ptr(q), ptr(pool.data), pool.pages, pool.shapes.page_bytes, ptr(tables), tables.stride(0),
            pool.fixed_pages, attn_layer, pool.shapes.attn_layers, ptr(pos), ptr(kn), ptr(vn), ptr(pr), pr.stride(0),
            ptr(y), y.stride(0), b, n)
    if scratch is None:
        _lib.call("jb_paged_attention_gated", *args, stream_ptr())
    else:
        _check(scratch, "attention scratch", torch.float32)
        _lib.call("jb_paged_attention_gated_split", *args, ptr(scratch), scratch.numel(), stream_ptr())
    return y


def kv_scatter(kn: torch.Tensor, vn: torch.Tensor, n: int, real: torch.Tensor, pool, out_tables: torch.Tensor,
               attn_layer: int) -> None:
    b = kn.shape[0] // n
    _lib.call("jb_kv_scatter", ptr(kn), ptr(vn), b, n, ptr(real), ptr(pool.data), pool.shapes.page_bytes,
              ptr(out_tables), out_tables.stride(0), pool.fixed_pages, attn_layer, pool.shapes.attn_layers,
              stream_ptr())


# ---------------------------------------------------------------- single tokens over the prefix pool


def _rows_of(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...], inner: int,
             device: torch.device) -> None:
    """`t` (shape) of `dtype` on `device`, its last `inner` dimensions packed and the others strided as they like."""
    if t.dtype is dtype and t.shape == shape and t.device == device and t.is_cuda and t.is_contiguous():
        return   # what nearly every call brings: these checks are most of a small call's host time
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: expected {dtype} of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device} as the others, got one on {t.device}")
    step = 1
    for size, stride in zip(reversed(shape[len(shape) - inner:]), reversed(t.stride()[len(shape) - inner:])):
        if stride != step and size != 1:
            raise ValueError(f"{name}: expected the last {inner} dimension(s) packed, got strides {t.stride()}")
        step *= size


def _tables_of(tables: torch.Tensor, name: str, rows: int, width: int, device: torch.device) -> None:
    """Block tables of at least `rows` rows and `width` entries, packed or with their rows apart. (The stride of a single
    row or page may be anything: the calls below give its packed size instead.)"""
    shape = tables.shape
    if len(shape) != 2 or shape[0] < rows or shape[1] < width or tables.dtype is not torch.int32 or \
            not (tables.is_contiguous() or tables.stride(1) == 1 or shape[1] == 1):
        raise ValueError(f"{name}: expected int32 (rows >= {rows}, width >= {width}) with packed rows, got "
                         f"{tuple(shape)} {tables.dtype}, strides {tables.stride()}")
    if tables.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got one on {tables.device}")


def _cache_of(kv: torch.Tensor, attn_layer: int, device: torch.device) -> torch.Size:
    """The shape of a cache of pages kv[page, layer, K|V, 32 tokens, head, dim]."""
    shape = kv.shape
    if len(shape) != 6 or shape[2] != 2 or shape[3] != 32:
        raise ValueError(f"kv: expected bf16 pages (page, layer, 2, 32, heads, dim), got {kv.dtype} {tuple(shape)}")
    _rows_of(kv, "kv", DT, shape, 5, device)
    if not 0 <= attn_layer < shape[1]:
        raise ValueError(f"attn_layer {attn_layer}: the pages hold {shape[1]} layers")
    return shape


def _on(device: torch.device, name: str, *args) -> None:
    """One library call on `device` and its current stream."""
    index = device.index
    # the stream's handle without a Stream object around it: 0.1 us on the host instead of 3.3
    if index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


class SlotMap(NamedTuple):
    """Where a pass's new tokens go (block_tables): per packed token its slot in the cache (page * page_tokens + place,
    -1 for none), its row and its position; each row's first token and the pages taken by the rows before it."""
    slots: torch.Tensor       # (tokens,) int64
    rows: torch.Tensor        # (tokens,) int32
    positions: torch.Tensor   # (tokens,) int32
    starts: torch.Tensor      # (b + 1,) int32
    taken: torch.Tensor       # (b + 1,) int32


def block_tables(lengths: torch.Tensor, new: torch.Tensor, free: torch.Tensor, tables: torch.Tensor, kv_entry: int,
                 tokens: int, *, page_tokens: int = 32, fixed: bool = False, out: SlotMap | None = None) -> SlotMap:
    """Block tables and slot maps from the requests' lengths, without the host. Row r holds lengths[r] tokens and adds
    new[r]; the pages its new tokens need come off `free` (int32 page ids, the first to take first) in row order and
    are written behind the row's own in `tables`, in place; fixed: a row that holds no token yet first takes kv_entry
    pages into its entries [0, kv_entry) (a prefix's state and convolution pages, PrefixPool.reserve's order). Every
    other entry stays as it was. `tokens` is the pass's capacity. taken[-1] > len(free) says that the free list was too
    short: the entries it leaves without a page name the sink (0), and their tokens' slots are -1, also those of later
    calls on these entries, as are those of tokens past the table's width. Page 0 is never a page to take: `free` must
    not list it."""
    dev = lengths.device
    b = lengths.shape[0] if lengths.dim() == 1 else -1
    _rows_of(lengths, "lengths", torch.int32, (b,), 1, dev)
    _rows_of(new, "new", torch.int32, (b,), 1, dev)
    if free.dim() != 1:
        raise ValueError(f"free: expected a vector of page ids, got {tuple(free.shape)}")
    _rows_of(free, "free", torch.int32, tuple(free.shape), 1, dev)
    _tables_of(tables, "tables", b, kv_entry + 1, dev)
    if out is None:
        parts = lengths.new_empty(4 * tokens + 2 * (b + 1)).split((2 * tokens, tokens, tokens, b + 1, b + 1))
        out = SlotMap(parts[0].view(torch.int64), *parts[1:])
    else:
        for name, dtype, size in (("slots", torch.int64, tokens), ("rows", torch.int32, tokens),
                                  ("positions", torch.int32, tokens), ("starts", torch.int32, b + 1),
                                  ("taken", torch.int32, b + 1)):
            _rows_of(getattr(out, name), name, dtype, (size,), 1, dev)
    slots, rows, positions, starts, taken = out
    width = tables.shape[1]
    _on(dev, "jb_block_tables", lengths.data_ptr(), new.data_ptr(), b, free.data_ptr(), free.shape[0],
        tables.data_ptr(), tables.stride(0) if b > 1 else width, width, kv_entry, page_tokens, 1 if fixed else 0,
        tokens, slots.data_ptr(), rows.data_ptr(), positions.data_ptr(), starts.data_ptr(), taken.data_ptr())
    return out


def rope_axes(sections: Sequence[int], interleaved: bool = False) -> int:
    """Which axis's position turns each of the 32 rotary frequencies, for attn_prep_axes: sections[a] frequencies of
    axis a, one axis after the other, or interleaved (frequency i belongs to axis i mod the number of axes while that
    axis has frequencies left, to axis 0 after that). At most four axes; 2 bits a frequency."""
    return _rope_axes(tuple(sections), interleaved)


@functools.lru_cache(maxsize=64)
def _rope_axes(sections: tuple[int, ...], interleaved: bool) -> int:
    n = len(sections)
    if not 1 <= n <= 4 or sum(sections) != C.ROT // 2 or min(sections) < 0:
        raise ValueError(f"sections {sections}: one to four axes with {C.ROT // 2} frequencies in all")
    if interleaved:
        of = [i % n if i // n < sections[i % n] else 0 for i in range(C.ROT // 2)]
    else:
        of = [a for a, count in enumerate(sections) for _ in range(count)]
    return sum(a << 2 * i for i, a in enumerate(of))


@functools.lru_cache(maxsize=64)
def _axes_fit(axes: int, count: int) -> bool:
    return 0 <= axes < 1 << C.ROT and all(axes >> 2 * i & 3 < count for i in range(C.ROT // 2))


def attn_prep_axes(pr: torch.Tensor, q_w1: torch.Tensor, k_w1: torch.Tensor, inv_freq: torch.Tensor,
                   positions: torch.Tensor, axes: int, *, kn: torch.Tensor | None = None,
                   vn: torch.Tensor | None = None, kv: torch.Tensor | None = None, attn_layer: int = 0,
                   slots: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """attn_prep_rows for any number of tokens, with positions (axes, t) int32 of several axes (axes from rope_axes;
    one axis: text). q (t, 8, 256); keys and values to kn and vn (t, 2, 256), into the cache pages kv at slots (t,)
    int64 (block_tables; -1: nowhere), or both. Two tokens must not have the same slot. Unlike attn_prep_rows, which
    keeps the reference's rounding points, everything between is fp32 (the angle fp64) and rounded once."""
    dev, t = pr.device, pr.shape[0]
    if pr.dim() != 2 or pr.shape[1] < C.ATTN_PROJ:
        raise ValueError(f"pr: expected (tokens, at least {C.ATTN_PROJ}), got {tuple(pr.shape)}")
    _rows_of(pr, "pr", DT, pr.shape, 1, dev)
    _rows_of(q_w1, "q_w1", torch.float32, (C.HD,), 1, dev)
    _rows_of(k_w1, "k_w1", torch.float32, (C.HD,), 1, dev)
    _rows_of(inv_freq, "inv_freq", torch.float32, (C.ROT // 2,), 1, dev)
    count = positions.shape[0] if positions.dim() == 2 else -1
    _rows_of(positions, "positions", torch.int32, (count, t), 1, dev)
    if not _axes_fit(axes, count):
        raise ValueError(f"axes: a frequency has an axis past the positions' {count}")
    for name, x in (("kn", kn), ("vn", vn)):
        if x is not None:
            _rows_of(x, name, DT, (t, C.NKV, C.HD), 3, dev)
    if slots is not None:
        _rows_of(slots, "slots", torch.int64, (t,), 1, dev)
    if kv is not None and _cache_of(kv, attn_layer, dev)[4:] != (C.NKV, C.HD):
        raise ValueError(f"kv: expected pages of {C.NKV} heads of {C.HD}, got {tuple(kv.shape)}")
    if out is None:
        out = pr.new_empty((t, C.NQ, C.HD))
    else:
        _rows_of(out, "out", DT, (t, C.NQ, C.HD), 3, dev)
    pages = (None, 0, 0, attn_layer, 0) if kv is None else (
        kv.data_ptr(), kv.shape[0], 2 * (kv.stride(0) if kv.shape[0] > 1 else kv.numel()), attn_layer, kv.shape[1])
    _on(dev, "jb_attn_prep_axes", pr.data_ptr(), pr.stride(0), t, q_w1.data_ptr(), k_w1.data_ptr(),
        inv_freq.data_ptr(), positions.data_ptr(), positions.stride(0), axes - (1 << 64) if axes >> 63 else axes,
        out.data_ptr(), ptr(kn), ptr(vn), *pages, ptr(slots))
    return out


@functools.lru_cache(maxsize=64)
def _decode_scratch(heads: int, kv_heads: int, dim: int) -> int:
    return _lib.load().jb_decode_attention_scratch(heads, kv_heads, dim)


def decode_attention(q: torch.Tensor, kv: torch.Tensor, tables: torch.Tensor, attn_layer: int, lengths: torch.Tensor,
                     kv_entry: int, *, scale: float | None = None, pr: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per row, q (b, heads, dim), over the row's lengths[r] cached tokens (its own among
    them, once attn_prep_axes has written it) in the pages tables[r][kv_entry + j // 32] of kv (an entry that is 0, the
    sink, or outside kv is no page: its tokens are left out); heads of 64, 128 or 256, up to 16 query heads to a
    key/value head, scale 1 / sqrt(dim) unless given. A row without tokens is zeros. What is not finite reaches what the
    formula lets it reach, an infinite value perhaps as NaN. With pr (the q_proj output, query and gate interleaved per
    head): times sigmoid(gate), as (b, heads * dim), the o_proj's input; without, (b, heads, dim). fp32 with one
    rounding. All rows' keys are cut into equal shares over the SMs, whatever the lengths; scratch (fp32,
    jb_decode_attention_scratch of them, overwritten by every call; calls that may run at the same time need their own)
    holds the cut rows' parts and is allocated unless given."""
    dev = q.device
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"q: expected (rows, heads, dim), got {tuple(shape)}")
    b, heads, dim = shape
    _rows_of(q, "q", DT, shape, 2, dev)
    pages, layers, _, _, kv_heads, kv_dim = _cache_of(kv, attn_layer, dev)
    if kv_dim != dim:
        raise ValueError(f"q: heads of {dim}, the pages' keys are {kv_dim} wide")
    _tables_of(tables, "tables", b, kv_entry, dev)
    _rows_of(lengths, "lengths", torch.int32, (b,), 1, dev)
    if pr is not None:
        if pr.dim() != 2 or pr.shape[1] < 2 * heads * dim:
            raise ValueError(f"pr: expected (rows, at least {2 * heads * dim}), got {tuple(pr.shape)}")
        _rows_of(pr, "pr", DT, (b, pr.shape[1]), 1, dev)
        shape = (b, heads * dim)
    if out is None:
        out = q.new_empty(shape)
    else:
        _rows_of(out, "out", DT, shape, len(shape) - 1, dev)
    if scratch is None:
        scratch = q.new_empty(_decode_scratch(heads, kv_heads, dim), dtype=torch.float32)
    else:
        _rows_of(scratch, "scratch", torch.float32, tuple(scratch.shape), scratch.dim(), dev)
    width = tables.shape[1]
    _on(dev, "jb_decode_attention", q.data_ptr(), q.stride(0), kv.data_ptr(), pages,
        2 * (kv.stride(0) if pages > 1 else kv.numel()), attn_layer, layers, tables.data_ptr(),
        tables.stride(0) if b > 1 else width, width, kv_entry, lengths.data_ptr(), b, heads, kv_heads, dim,
        dim ** -0.5 if scale is None else scale, ptr(pr), 0 if pr is None else pr.stride(0),
        out.data_ptr(), out.stride(0), scratch.data_ptr(), scratch.numel())
    return out


# ---------------------------------------------------------------- linear attention with a decay for each head


def _linear_of(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
               tables: torch.Tensor, layer: int, out_tables: torch.Tensor | None,
               out: torch.Tensor | None) -> tuple[torch.Tensor, tuple]:
    """What linear_scan and linear_step check alike; (o, the states' arguments)."""
    dev, shape = q.device, q.shape
    b, heads = shape[0], shape[-2]
    if shape[-1] != C.DK:
        raise ValueError(f"q: expected heads of {C.DK}, got {tuple(shape)}")
    if not (q.shape == shape and k.shape == shape and v.shape == shape and q.dtype is DT and k.dtype is DT and
            v.dtype is DT and q.is_cuda and k.device == dev and v.device == dev and q.is_contiguous() and
            k.is_contiguous() and v.is_contiguous()):
        for name, x in (("q", q), ("k", k), ("v", v)):
            _rows_of(x, name, DT, shape, 2, dev)
    if g.dim() == 1:
        _rows_of(g, "g", torch.float32, (heads,), 1, dev)
    else:
        _rows_of(g, "g", torch.float32, shape[:-1], 1, dev)
    held = state.shape
    if len(held) != 4 or held[2:] != (C.DK, C.DV):
        raise ValueError(f"state: expected pages (page, heads per page, {C.DK}, {C.DV}), got {tuple(held)}")
    _rows_of(state, "state", torch.float32, held, 3, dev)
    if layer < 0:
        raise ValueError(f"layer {layer}: layers count from 0")
    width = (layer * heads + heads - 1) // held[1] + 1
    _tables_of(tables, "tables", b, width, dev)
    if out_tables is not None and out_tables is not tables:
        _tables_of(out_tables, "out_tables", b, width, dev)
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    else:
        _rows_of(out, "out", DT, shape, len(shape), dev)
    one = b == 1
    return out, (state.data_ptr(), held[0], 4 * (state.stride(0) if held[0] > 1 else state.numel()), held[1],
                 layer * heads, tables.data_ptr(), width if one else tables.stride(0), ptr(out_tables),
                 0 if out_tables is None else width if one else out_tables.stride(0))


@functools.lru_cache(maxsize=256)
def _scan_scratch(b: int, heads: int, n: int) -> int:
    return _lib.load().jb_linear_scan_scratch(b, heads, n)


def linear_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                tables: torch.Tensor, layer: int, *, real: torch.Tensor | None = None,
                out_tables: torch.Tensor | None = None, out: torch.Tensor | None = None,
                scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Linear attention with a decay for each head over q, k, v (b, n, heads, 128): S_t = e^g S_(t-1) + k_t v_t^T, o_t =
    S_t^T q_t / sqrt(128), each row from its state in the pages `state` (PrefixPool.state; head h of `layer` is flat
    head layer * heads + h) that its row of tables names. g: log-decays (b, n, heads) fp32, or (heads,), one for each
    head; -inf forgets. real (b,) int32: row r has real[r] tokens, its outputs past them are zeros. out_tables: the
    rows' final states are written to these pages (the reserved pages 0 and 1 never are); rows must not share them, nor
    write pages that another row reads. A state on page 0, the sink, or outside `state` reads as zeros. scratch (fp32,
    jb_linear_scan_scratch of them, one for each of the calls that may run at the same time) is allocated unless given.
    What is not finite in q, k, v, g or a state spoils what the recurrence spoils, no earlier output and no other head;
    where that gives an infinity it may be NaN. out must not overlap q, k or v."""
    if q.dim() != 4:
        raise ValueError(f"q: expected (rows, tokens, heads, {C.DK}), got {tuple(q.shape)}")
    b, n, heads = q.shape[:3]
    o, pool = _linear_of(q, k, v, g, state, tables, layer, out_tables, out)
    if real is not None:
        _rows_of(real, "real", torch.int32, (b,), 1, q.device)
    need = _scan_scratch(b, heads, n)
    (q0, q1, _, _), (k0, k1, _, _), (v0, v1, _, _) = q.stride(), k.stride(), v.stride()
    if need and not (q1 and k1 and v1 and (b == 1 or q0 and k0 and v0)):
        need = 0   # one token or row that stands for all goes token by token, in one launch
    if scratch is None:
        scratch = q.new_empty(need, dtype=torch.float32) if need else None
    else:
        _rows_of(scratch, "scratch", torch.float32, tuple(scratch.shape), scratch.dim(), q.device)
    steps = (0, 0) if g.dim() == 1 else g.stride()[:2]
    _on(q.device, "jb_linear_scan", q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, g.data_ptr(),
        *steps, ptr(real), o.data_ptr(), b, n, heads, *pool, ptr(scratch), 0 if scratch is None else scratch.numel())
    if need:
        _lib.launches += 2   # in segments: their states, the join, the outputs
    return o


def linear_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                tables: torch.Tensor, layer: int, *, beta: torch.Tensor | None = None,
                out_tables: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """linear_scan's recurrence for one token per row, q, k, v (b, heads, 128), g (b, heads) or (heads,): o (b, heads,
    128), the new states written in place, or to out_tables' pages (rows must not share them, nor write pages that
    another row reads; the new state of a row whose page is 0 or 1, reserved, is dropped). beta (b, heads) bf16: the
    gated delta rule of gdn_scan, v replaced by beta (v - (e^g S)^T k). out must not overlap q, k or v."""
    if q.dim() != 3:
        raise ValueError(f"q: expected (rows, heads, {C.DK}), got {tuple(q.shape)}")
    b, heads = q.shape[:2]
    o, pool = _linear_of(q, k, v, g, state, tables, layer, tables if out_tables is None else out_tables, out)
    if beta is not None:
        _rows_of(beta, "beta", DT, (b, heads), 2, q.device)
    _on(q.device, "jb_linear_step", q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
        g.data_ptr(), 0 if g.dim() == 1 else g.stride(0), ptr(beta), o.data_ptr(), b, heads, *pool)
    return o
