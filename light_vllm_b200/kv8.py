"""A paged K/V cache held in 8 bits, and attention over it.

Codes of one byte (``torch.int8`` or ``torch.float8_e4m3fn``) with one fp32
scale for each block and KV head, for the keys and for the values: half the
bytes of the 16-bit cache (runtime/execution/paged_cache.py:30-338, which has no
8-bit form), so twice the context fits.  A decode step reads half as much, and is
about a tenth faster: 64 requests of 512 to 4096 tokens, 28/4 heads of 128, bf16,
53.8 us (append 3.2, attention 49.6) beside the 16-bit cache's 60.5 us with its
write.

* ``kv8_append`` -- rotate a step's queries and keys and append its keys and
  values (``lvb_kv8_append``);
* ``kv8_attention`` -- attention of the step's packed queries over the cache
  (``lvb_kv8_attention``): single tokens, drafts under verification, prompt
  chunks, any mix;
* ``kv8_read_blocks`` -- values of whole blocks in the model's type
  (``lvb_kv8_read_blocks``);
* ``KV8Cache`` and ``B200KV8AttentionBackend`` -- the same behind the contract
  of ``PagedAttentionBackend`` (runtime/execution/paged_attention.py:209-223):
  a step's attention context for ``Qwen2AWQRunner`` or a ``ForwardBatch``.

A block's scales only grow while the block is filled, drafted tokens that are
refused later included: their slots are written over by the next step, but the
step of the codes stays what the largest value needed.

All of it runs on the current stream, allocates through torch and does not
synchronise.  A call goes through ``_torch_ops`` (``csrc/torch_ops.cpp``), which
checks and launches the usual case; the functions below hold every rule and
message and take whatever that hands back.
"""

from __future__ import annotations

from collections.abc import Iterable
from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch import Tensor

from light_vllm_b200 import _native
from light_vllm_b200.kv_cache import KVCacheError
from light_vllm_b200.paged_attention import StepMetadataPacker
from light_vllm_b200.staging import SingleStepStaging

_ACT_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}
_CODE_DTYPES = {torch.int8: _native.KV8_INT8, torch.float8_e4m3fn: _native.KV8_E4M3}


class KV8Layer(NamedTuple):
    """One layer's cache: codes [num_blocks, kv_heads, block_size, head_size]
    and fp32 scales [num_blocks, kv_heads], all contiguous."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor
    value_scales: Tensor


class KV8Step(NamedTuple):
    """A step's packed requests: int32 tensors on the device as
    ``lvb_pack_step_metadata`` lays them out, and two host numbers.
    ``max_query_len`` is the longest request's query count, ``max_seq_len`` the
    longest context (computed and query tokens), which bounds nothing."""

    block_tables: Tensor  # [requests, blocks], rows at any stride
    num_computed: Tensor  # [requests], tokens cached by earlier steps
    query_start: Tensor  # [requests + 1], prefix sums of query lengths
    max_query_len: int
    max_seq_len: int


def _check_layer(layer: KV8Layer) -> int:
    """The layer's code type; raises ``KVCacheError`` for a malformed layer."""

    keys, values, key_scales, value_scales = layer
    code = _CODE_DTYPES.get(keys.dtype)
    if code is None or values.dtype != keys.dtype:
        raise KVCacheError("KV8 codes must be int8 or float8_e4m3fn, keys and values alike")
    shape = keys.shape
    if len(shape) != 4 or values.shape != shape:
        raise KVCacheError("KV8 codes must be [num_blocks, kv_heads, block_size, head_size]")
    if (key_scales.dtype != torch.float32 or value_scales.dtype != torch.float32
            or key_scales.shape != shape[:2] or value_scales.shape != shape[:2]):
        raise KVCacheError("KV8 scales must be float32 [num_blocks, kv_heads]")
    if not (keys.is_contiguous() and values.is_contiguous() and key_scales.is_contiguous()
            and value_scales.is_contiguous()):
        raise KVCacheError("KV8 codes and scales must be contiguous")
    device = keys.get_device()
    if (device < 0 or values.get_device() != device or key_scales.get_device() != device
            or value_scales.get_device() != device):
        raise KVCacheError("KV8 codes and scales must share one CUDA device")
    return code


def _check_step(step: KV8Step, device: int) -> int:
    """The number of requests; raises ``KVCacheError`` for a malformed step."""

    tables, computed, start = step[:3]
    n = computed.shape[0] if len(computed.shape) == 1 else -1
    if (n < 0 or tables.dtype != torch.int32 or computed.dtype != torch.int32 or start.dtype != torch.int32
            or len(tables.shape) != 2 or tables.shape[0] != n or start.shape != (n + 1,)):
        raise KVCacheError("KV8 step metadata must be int32 [n, blocks], [n] and [n + 1]")
    if (tables.get_device() != device or computed.get_device() != device or start.get_device() != device):
        raise KVCacheError("KV8 step metadata must be on the cache's device")
    if not computed.is_contiguous() or not start.is_contiguous() or (tables.shape[1] > 1 and tables.stride(1) != 1):
        raise KVCacheError("KV8 step metadata must be contiguous")
    return n


def _check_rows(name: str, rows: Tensor, tokens: int, heads: int | None, head_size: int, dtype: torch.dtype,
                device: int) -> None:
    shape = rows.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_size or (heads is not None and shape[1] != heads):
        raise KVCacheError(f"KV8 {name} rows must be [tokens, heads, head_size] of the cache's heads")
    if rows.dtype != dtype or rows.get_device() != device:
        raise KVCacheError(f"KV8 {name} rows must share one dtype (fp16 or bf16) and the cache's device")


def _dense_heads(rows: Tensor) -> Tensor:
    """Rows whose heads are dense and in order (a token's stride is free)."""

    tokens, heads, d = rows.shape
    if rows.is_contiguous() or (rows.stride(2) == 1 and (heads == 1 or rows.stride(1) == d)
                                and (tokens == 1 or rows.stride(0) >= heads * d)):
        return rows
    return rows.contiguous()


def _token_stride(rows: Tensor) -> int:
    """Elements from token to token; a single one's stride means nothing (torch
    keeps whatever its storage had), so it is what the heads take."""

    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1] * rows.shape[2]


class _Workspaces:
    """Scratch of one operator, zero where its calls want it and left so by them: a
    buffer for each (device, stream), whose calls follow one another, and for
    each capture a buffer of its own in the graph's memory, zeroed by the graph,
    since a graph may be replayed on any stream, beside whatever runs there."""

    def __init__(self, op: int, zero_bytes: int | None = None) -> None:
        self._op = op
        self._zero_bytes = zero_bytes  # that have to be zero (None: all of it)
        self._current: dict[tuple[int, int], Tensor] = {}
        self._captured: dict[tuple[int, int], tuple[int, Tensor]] = {}

    def get(self, device: torch.device, stream: int, need: int) -> tuple[int, int]:
        if need == 0:
            return 0, 0
        key = (device.index, stream)
        capture = _native.stream_capture_id(stream)
        if capture:
            held, buf = self._captured.get(key, (0, None))
            if held != capture or buf.numel() < need:
                buf = torch.empty(need, dtype=torch.uint8, device=device)
                buf[:self._zero_bytes].zero_()
                # (former captures' buffers go back to their graphs' memory)
                self._captured = {k: v for k, v in self._captured.items() if v[0] == capture}
                self._captured[key] = capture, buf
            return buf.data_ptr(), buf.numel()
        buf = self._current.get(key)
        if buf is None or buf.numel() < need:
            buf = torch.zeros(max(1 << 20, 1 << (need - 1).bit_length()), dtype=torch.uint8, device=device)
            self._current[key] = buf
            _native.torch_ops().set_scratch(self._op, device.index, stream, buf.data_ptr(), buf.numel())
        return buf.data_ptr(), buf.numel()


_workspaces = _Workspaces(0, _native.KV8_COUNTER_BYTES)
_fast = None  # _torch_ops, loaded by the first call


def _ops():
    global _fast
    if _fast is None:
        _fast = _native.torch_ops()
    return _fast


def kv8_append(query: Tensor | None, key: Tensor, value: Tensor, layer: KV8Layer, step: KV8Step, *,
               positions: Tensor | None = None, cos: Tensor | None = None, sin: Tensor | None = None,
               query_out: Tensor | None = None) -> Tensor | None:
    """Append the step's key and value rows [tokens, kv_heads, head_size] to
    ``layer`` and return the rotated query rows [tokens, heads, head_size].

    With ``positions`` (int32, one for each token) and the tables ``cos`` /
    ``sin`` [rows, head_size] of the rows' dtype, queries and keys are rotated
    as ``lvb_rope_qk`` does; the keys go into the cache without a rounding
    between.  Without them keys are appended as they are, and ``query`` must be
    None.  ``query_out`` (``query`` itself, if wanted) receives the rotated
    queries instead of a new tensor."""

    done = (_fast or _ops()).kv8_append(query, key, value, *layer, *step, positions, cos, sin, query_out)
    if done is not None:
        if type(done) is int:
            _native.check(done, "lvb_kv8_append")
        return None if done is True else done
    code = _check_layer(layer)
    keys = layer.keys
    num_blocks, hkv, block, d = keys.shape
    device = keys.device
    index = device.index
    n = _check_step(step, index)
    dtype = key.dtype
    act = _ACT_DTYPES.get(dtype)
    if act is None:
        raise KVCacheError("KV8 rows must be fp16 or bf16")
    tokens = key.shape[0] if key.dim() else 0
    _check_rows("key", key, tokens, hkv, d, dtype, index)
    _check_rows("value", value, tokens, hkv, d, dtype, index)
    key, value = _dense_heads(key), _dense_heads(value)
    pos_ptr = cos_ptr = sin_ptr = table_rows = q_ptr = q_stride = out_ptr = out_stride = hq = 0
    if positions is not None:
        if cos is None or sin is None:
            raise KVCacheError("KV8 rotation needs the cos and sin tables")
        if (positions.dtype != torch.int32 or positions.shape != (tokens,) or positions.get_device() != index
                or not positions.is_contiguous()):
            raise KVCacheError("KV8 positions must be int32, one for each token, on the cache's device")
        if (cos.shape != sin.shape or len(cos.shape) != 2 or cos.shape[1] != d or cos.dtype != dtype
                or sin.dtype != dtype or cos.get_device() != index or sin.get_device() != index
                or not cos.is_contiguous() or not sin.is_contiguous()):
            raise KVCacheError("KV8 rotation tables must be [rows, head_size] of the rows' dtype and device")
        pos_ptr, cos_ptr, sin_ptr, table_rows = positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    if query is not None:
        if positions is None:
            raise KVCacheError("KV8 queries are only rotated: pass positions, or no query")
        _check_rows("query", query, tokens, None, d, dtype, index)
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=dtype, device=device)
        else:
            _check_rows("query output", query_out, tokens, query.shape[1], d, dtype, index)
            if _dense_heads(query_out) is not query_out:
                raise KVCacheError("KV8 query output rows must have dense heads")
        query = _dense_heads(query)
        hq = query.shape[1]
        q_ptr, q_stride, out_ptr, out_stride = (query.data_ptr(), _token_stride(query), query_out.data_ptr(),
                                                _token_stride(query_out))
    if tokens and n:
        with _on(index):
            _native.check(_native.library().lvb_kv8_append_strided(
                q_ptr, q_stride, out_ptr, out_stride, key.data_ptr(), _token_stride(key), value.data_ptr(),
                _token_stride(value), pos_ptr, cos_ptr, sin_ptr, table_rows, keys.data_ptr(), layer.values.data_ptr(),
                layer.key_scales.data_ptr(), layer.value_scales.data_ptr(), step.block_tables.data_ptr(),
                step.block_tables.shape[1], step.block_tables.stride(0), step.num_computed.data_ptr(), step.query_start.data_ptr(), n, tokens,
                step.max_query_len, hq, hkv, d, block, num_blocks, act, code, _native.stream_handle(device)),
                "lvb_kv8_append")
    return query_out


def kv8_read_blocks(layer: KV8Layer, block_ids: Tensor, *, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    """Keys and values [n, kv_heads, block_size, head_size] of the blocks
    ``block_ids`` (int32 on the cache's device) in ``dtype``."""

    act = _ACT_DTYPES.get(dtype)
    if act is not None:
        done = (_fast or _ops()).kv8_read_blocks(*layer, block_ids, dtype is torch.bfloat16)
        if done is not None:
            if type(done) is int:
                _native.check(done, "lvb_kv8_read_blocks")
            return done
    code = _check_layer(layer)
    if act is None:
        raise KVCacheError("KV8 blocks are read in fp16 or bf16")
    keys = layer.keys
    num_blocks, hkv, block, d = keys.shape
    device = keys.device
    if (block_ids.dtype != torch.int32 or len(block_ids.shape) != 1 or block_ids.get_device() != device.index
            or not block_ids.is_contiguous()):
        raise KVCacheError("KV8 block ids must be a contiguous int32 vector on the cache's device")
    n = block_ids.shape[0]
    out = torch.empty((2, n, hkv, block, d), dtype=dtype, device=device)
    key_out, value_out = out[0], out[1]
    if n:
        with _on(device.index):
            _native.check(_native.library().lvb_kv8_read_blocks(
                keys.data_ptr(), layer.values.data_ptr(), layer.key_scales.data_ptr(), layer.value_scales.data_ptr(),
                block_ids.data_ptr(), n, key_out.data_ptr(), value_out.data_ptr(), hkv, d, block, num_blocks, act,
                code, _native.stream_handle(device)), "lvb_kv8_read_blocks")
    return key_out, value_out


def kv8_attention(query: Tensor, layer: KV8Layer, step: KV8Step, *, scale: float, out: Tensor | None = None) -> Tensor:
    """Attention of the step's query rows [tokens, heads, head_size] over
    ``layer``, which must hold the step's own tokens already: token t of a
    request sees every position up to its own.  ``out`` receives the result
    instead of a new tensor; rows of no request, or of one that the device
    refuses, are left as they are.

    Scores, softmax statistics and sums are fp32; the weights enter the second
    product as fp16 (11 bits), bf16 queries the first as fp16 times a power of
    two (exact down to 2^-22 of the row's largest element)."""

    done = (_fast or _ops()).kv8_attention(query, *layer, *step, scale, out)
    if done is not None:
        if type(done) is int:
            _native.check(done, "lvb_kv8_attention")
        return done
    code = _check_layer(layer)
    keys = layer.keys
    num_blocks, hkv, block, d = keys.shape
    device = keys.device
    index = device.index
    n = _check_step(step, index)
    dtype = query.dtype
    act = _ACT_DTYPES.get(dtype)
    if act is None:
        raise KVCacheError("KV8 rows must be fp16 or bf16")
    tokens = query.shape[0] if query.dim() else 0
    _check_rows("query", query, tokens, None, d, dtype, index)
    hq = query.shape[1]
    if hq == 0 or hq % hkv:
        raise KVCacheError("KV8 query heads must be a multiple of the KV heads")
    if out is None:
        out = torch.empty(query.shape, dtype=dtype, device=device)
    else:
        _check_rows("output", out, tokens, hq, d, dtype, index)
        if _dense_heads(out) is not out or out.data_ptr() % 16 or _token_stride(out) % 8:
            raise KVCacheError("KV8 output rows must have dense heads and be 16-byte aligned")
    query = _dense_heads(query)
    if query.data_ptr() % 16 or _token_stride(query) % 8:
        query = query.clone(memory_format=torch.contiguous_format)
    if tokens and n:
        with _on(index):
            lib = _native.library()
            stream = _native.stream_handle(device)
            need = lib.lvb_kv8_attention_workspace_bytes(n, hq, hkv, d, step.max_query_len, step.max_seq_len)
            ws, ws_bytes = _workspaces.get(device, stream, need)
            _native.check(lib.lvb_kv8_attention_strided(
                query.data_ptr(), _token_stride(query), keys.data_ptr(), layer.values.data_ptr(),
                layer.key_scales.data_ptr(), layer.value_scales.data_ptr(), out.data_ptr(), _token_stride(out),
                step.block_tables.data_ptr(), step.block_tables.shape[1], step.block_tables.stride(0),
                step.num_computed.data_ptr(), step.query_start.data_ptr(), n, tokens, step.max_query_len, step.max_seq_len, hq, hkv, d, block,
                num_blocks, scale, act, code, ws, ws_bytes, stream), "lvb_kv8_attention")
    return out


class _Same:
    def __enter__(self) -> None:
        return None

    def __exit__(self, *exc) -> None:
        return None


_SAME = _Same()


def _on(index: int):
    """The tensors' device made current (launches go to the current device)."""

    return _SAME if torch.cuda.current_device() == index else torch.cuda.device(index)


class KV8LayerSpec(NamedTuple):
    """One attention layer's heads on this rank (``Qwen2AWQRunner.kv_layers()``)."""

    layer_id: str
    num_query_heads: int
    num_kv_heads: int
    head_size: int


@dataclass(frozen=True, slots=True)
class KV8CacheConfig:
    """Geometry of a ``KV8Cache``; ``dtype`` is the type of its codes."""

    num_blocks: int
    block_size: int
    dtype: torch.dtype = torch.int8
    device: str | torch.device = "cuda"

    def __post_init__(self) -> None:
        if type(self.num_blocks) is not int or self.num_blocks <= 0:
            raise ValueError("num_blocks must be a positive integer")
        if type(self.block_size) is not int or self.block_size <= 0 or self.block_size % 16 or self.block_size > 1024:
            raise ValueError("an 8-bit KV cache's block_size must be a multiple of 16 up to 1024")
        if self.dtype not in _CODE_DTYPES:
            raise ValueError("an 8-bit KV cache's dtype must be int8 or float8_e4m3fn")
        object.__setattr__(self, "device", torch.device(self.device))


class KV8Cache:
    """The 8-bit counterpart of ``PagedKVCache``
    (runtime/execution/paged_cache.py:328-338): zero-filled codes and scales of
    every layer, reached through ``layer(layer_id)``.  Rows may be fp16 or bf16.

    ``layers`` are (layer_id, query heads, KV heads, head size), as
    ``Qwen2AWQRunner.kv_layers()`` gives them.  ``compact_kv`` does not take this
    cache: accepted drafts of a linear layout need no move."""

    def __init__(self, layers: Iterable[tuple[str, int, int, int]], config: KV8CacheConfig) -> None:
        self.config = config
        self._specs = {spec[0]: KV8LayerSpec(*spec) for spec in layers}
        self._layers: dict[str, KV8Layer] = {}
        for spec in self._specs.values():
            if spec.head_size not in (64, 128):
                raise ValueError("an 8-bit KV cache's head sizes are 64 and 128")
            if spec.num_kv_heads <= 0 or spec.num_query_heads <= 0 or spec.num_query_heads % spec.num_kv_heads:
                raise ValueError("num_query_heads must be a positive multiple of num_kv_heads")
            codes = (config.num_blocks, spec.num_kv_heads, config.block_size, spec.head_size)
            self._layers[spec.layer_id] = KV8Layer(
                *(torch.zeros(codes, dtype=config.dtype, device=config.device) for _ in range(2)),
                *(torch.zeros(codes[:2], dtype=torch.float32, device=config.device) for _ in range(2)))

    @property
    def layer_ids(self) -> tuple[str, ...]:
        return tuple(self._specs)

    def layer_spec(self, layer_id: str) -> KV8LayerSpec:
        try:
            return self._specs[layer_id]
        except KeyError:
            raise KVCacheError(f"unknown attention layer {layer_id!r}") from None

    def layer(self, layer_id: str) -> KV8Layer:
        self.layer_spec(layer_id)
        return self._layers[layer_id]


class B200KV8Attention:
    """Per-step attention context over a ``KV8Cache``; one ``forward`` per layer.
    ``step`` is the step's packed metadata."""

    def __init__(self, cache: KV8Cache, step: KV8Step, num_tokens: int) -> None:
        self.step = step
        self._cache = cache
        self._num_tokens = num_tokens
        self._layer_ids: set[str] = set()

    @property
    def layer_ids(self) -> frozenset[str]:
        return frozenset(self._layer_ids)

    def forward(self, layer_id: str, query: Tensor, key: Tensor, value: Tensor, *, scale: float,
                write_kv: bool = True) -> Tensor:
        """Append this step's K/V to ``layer_id`` and return the attention output.

        ``write_kv=False``: they are already in the cache (``rope_write_kv``)."""

        if layer_id in self._layer_ids:
            raise KVCacheError(f"paged attention layer {layer_id!r} ran more than once")
        spec = self._cache.layer_spec(layer_id)
        # The shape rules of the 16-bit backend (paged_attention.py:226-247).
        if query.dim() != 3:
            raise KVCacheError("paged attention query must have three dimensions")
        if query.shape[0] != key.shape[0] or value.shape != key.shape:
            raise KVCacheError("paged attention Q/K/V token dimensions must match")
        if query.shape[0] != self._num_tokens:
            raise KVCacheError("paged attention metadata token count does not match query")
        if query.shape[1:] != (spec.num_query_heads, spec.head_size):
            raise KVCacheError("paged attention query shape does not match the layer spec")
        if key.shape[1:] != (spec.num_kv_heads, spec.head_size):
            raise KVCacheError("paged attention K/V shape does not match the layer spec")
        self._layer_ids.add(layer_id)
        layer = self._cache.layer(layer_id)
        if write_kv:
            kv8_append(None, key, value, layer, self.step)
        return kv8_attention(query, layer, self.step, scale=float(scale))

    def rope_write_kv(self, layer_id: str, qkv: Tensor, q_heads: int, kv_heads: int, positions: Tensor,
                      cos: Tensor, sin: Tensor) -> None:
        """Rotate the query heads of merged QKV rows in place and append the
        rotated keys and the values to ``layer_id``; follow with
        ``forward(..., write_kv=False)``.  The key rows stay as they are."""

        spec = self._cache.layer_spec(layer_id)
        d = spec.head_size
        if ((q_heads, kv_heads) != (spec.num_query_heads, spec.num_kv_heads) or qkv.dim() != 2
                or qkv.shape != (self._num_tokens, (q_heads + 2 * kv_heads) * d)):
            raise KVCacheError("QKV heads or tokens do not match the layer")
        heads = qkv.unflatten(1, (-1, d))
        query = heads[:, :q_heads]
        kv8_append(query, heads[:, q_heads:q_heads + kv_heads], heads[:, q_heads + kv_heads:],
                   self._cache.layer(layer_id), self.step, positions=positions, cos=cos, sin=sin, query_out=query)


class B200KV8AttentionBackend:
    """Creates one ``B200KV8Attention`` per model step, from light-vllm's own
    ``PagedAttentionMetadata`` (linear layouts: a tree's rows see other positions
    than their prefix).  The metadata is checked, packed and copied to the
    device as ``B200PagedAttentionBackend`` does; the block-table rules and
    their messages are the same."""

    name = "b200-kv8"

    def __init__(self) -> None:
        _native.library()  # fail loudly at construction when the library is missing
        self._packer = StepMetadataPacker()
        self._staging: dict[torch.device, SingleStepStaging] = {}

    def create(self, cache: KV8Cache, metadata) -> B200KV8Attention:
        config = cache.config
        device = config.device
        if device.type != "cuda":
            raise KVCacheError("B200 paged attention requires a CUDA KV cache")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        shape = self._packer.gather(metadata)
        if not shape.linear:
            raise KVCacheError("the 8-bit KV cache covers linear query layouts")
        staging = self._staging.get(device)
        if staging is None:
            staging = self._staging[device] = SingleStepStaging(device)
        packed = self._packer.stage(staging, config.num_blocks, config.block_size)
        n, width = shape.num_seqs, shape.max_blocks
        tables, computed, start = packed[:n * (width + 2) + 1].split((n * width, n, n + 1))
        step = KV8Step(tables.view(n, width), computed, start, shape.max_query_len, shape.max_seq_len)
        return B200KV8Attention(cache, step, shape.num_tokens)
