"""The operators around the MLP of a decode step: attention over a paged cache, the cache's new slots,
the norms and the residual between two blocks, and the pick of the next tokens.

Each class binds the tensors of one call (the cold path: checks, the argument block, a workspace) and
`enqueue` puts the call on a stream as often as wanted; a decode loop keeps its buffers and refills
them. Definitions, limits and the meaning of every argument: include/leanstream_hip.h
(ls_hip_attention, ls_hip_append, ls_hip_block_norm, ls_hip_sample). Tensors are on the GPU and their
last dimension is contiguous; every other stride is free within those limits. Bad arguments raise
ValueError or, where the library refuses them, RuntimeError.

    cache = PagedCache(k_pages, v_pages)              # [pages, kv_heads, page_size, head_dim]
    append = AppendKV(q, k, v, cos, sin, cache, page_table, q_start, context, q_rotated)
    attention = PagedAttention(q_rotated, cache, page_table, q_start, context, out, max_new=1, max_context=8192)
    norm = BlockNorm(block, residual, hidden, normed, pre_weight=weight)
    sampler = Sampler(logits, uniform, tokens, temperature=temperature, top_p=top_p)
    for call in (append, attention, norm, sampler):
        call.enqueue()
"""
import ctypes as C
import functools

from . import _native
from .backend import _ptr

TYPES = {"torch.float16": 0, "torch.bfloat16": 1, "torch.float32": 2}


def _check(tensor, name, shape=None, dtype=None, optional=False):
    if tensor is None:
        if optional:
            return
        raise ValueError(f"{name} is missing")
    if not tensor.is_cuda:
        raise ValueError(f"{name} is not on the GPU")
    if dtype is not None and str(tensor.dtype) != dtype:
        raise ValueError(f"{name} is {tensor.dtype}, not {dtype}")
    if shape is not None and tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(tensor.shape)}, not {tuple(shape)}")
    if tensor.dim() and tensor.shape[-1] > 1 and tensor.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension is not contiguous")


def _dtype(tensor, name):
    if str(tensor.dtype) not in TYPES:
        raise ValueError(f"{name} is {tensor.dtype}: float16, bfloat16 or float32 expected")
    return TYPES[str(tensor.dtype)]


def _stride(tensor, dim):
    """Elements from one index to the next; 0 where there is only one, whose stride may be anything."""
    return tensor.stride(dim) if tensor.shape[dim] > 1 else 0


class _Call:
    """One bound call: the argument block, the tensors it points into, and the entry point."""

    def _bind(self, name, block, keep, workspace=None):
        lib = _native.library()
        self.name, self.block, self._keep = name, block, keep
        self._enqueue = getattr(lib, f"ls_hip_{name}_enqueue")
        self._arg = C.byref(block)
        self._device = next(t for t in keep if t is not None).device
        import torch

        if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
            raise ValueError("workspace is a contiguous tensor of bytes")
        if any(t.device != self._device for t in (*keep, workspace) if t is not None):
            raise ValueError(f"tensors on more than one device, or off the GPU: {self._device} expected")

        # the handle alone: torch.cuda.current_stream() makes an object of it first, 1.9 us of a 3.5 us call
        self._current = functools.partial(torch._C._cuda_getCurrentRawStream, self._device.index)
        self._current_device = torch._C._cuda_getDevice
        need = int(getattr(lib, f"ls_hip_{name}_workspace")(self._arg)) if hasattr(block, "workspace") else 0
        self._streams = None    # those in order with a workspace of the call's own
        if need and workspace is None and torch.cuda.is_current_stream_capturing():
            if name == "attention":     # its zeros would be part of the graph, and missing outside
                raise RuntimeError("attention needs a workspace: bind it before the capture, or hand one in")
            workspace = torch.empty(need, dtype=torch.uint8, device=self._device)
        elif need and workspace is None:
            with torch.cuda.device(self._device):
                workspace = torch.zeros(need, dtype=torch.uint8, device=self._device)
                self._zeroed = torch.cuda.Event()
                self._zeroed.record()
            self._streams = {self._current()}
        if workspace is not None:
            block.workspace, block.workspace_bytes = workspace.data_ptr(), workspace.numel()
        self.workspace = workspace

    def enqueue(self, stream=None):
        """Put the call on `stream` (a hipStream_t handle; default: torch's current stream). A stream handed in
        outlives the call, unless the call's workspace was handed in too."""
        if stream is None:
            stream = self._current()
        if self._streams is not None and stream not in self._streams:
            self._join(getattr(stream, "value", stream) or 0)
        if self._current_device() == self._device.index:
            rc = self._enqueue(self._arg, stream)
        else:       # the default stream's handle is 0 on every device: a launch goes to the current one
            import torch

            with torch.cuda.device(self._device):
                rc = self._enqueue(self._arg, stream)
        if rc:
            raise RuntimeError(f"Native {self.name} failed: {rc}")

    def _join(self, handle):
        """The caller does not see that the call's own workspace is zeroed on the stream on which it was bound, nor when it
        is freed: another stream waits for the one, and the other waits for that stream's work."""
        import torch

        stream = torch.cuda.ExternalStream(handle, self._device) if handle else torch.cuda.default_stream(self._device)
        if self._zeroed.query():
            self._streams.add(handle)
        else:
            with torch.cuda.stream(stream):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(f"{self.name}: wait for the stream on which it was bound before the capture")
            stream.wait_event(self._zeroed)
        self.workspace.record_stream(stream)


class PagedCache:
    """Keys and values of all sequences in pages: two tensors [pages, kv_heads, page_size, head_dim] of
    any stride order (contiguous, a page's keys of one head lie in one piece)."""

    def __init__(self, k, v):
        _check(k, "k")
        _check(v, "v", k.shape, str(k.dtype))
        if k.dim() != 4:
            raise ValueError("pages have the dimensions [pages, kv_heads, page_size, head_dim]")
        self.k, self.v = k, v
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, dtype, device="cuda"):
        import torch

        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def _check_sequences(page_table, q_start, context, status):
    _check(page_table, "page_table", dtype="torch.int32")
    if page_table.dim() != 2:
        raise ValueError("page_table has the dimensions [sequences, pages of a sequence]")
    _check(q_start, "q_start", (page_table.shape[0] + 1,), "torch.int32")
    _check(context, "context", (page_table.shape[0],), "torch.int32")
    _check(status, "status", dtype="torch.int32", optional=True)


class PagedAttention(_Call):
    """out [tokens, q_heads, head_dim]: attention of the new tokens q over their sequences' keys in `cache`.
    max_new and max_context bound a sequence's new tokens and keys; scale (> 0) defaults to head_dim ** -0.5;
    window and sinks restrict a token to its last `window` keys and the sequence's first `sinks`. lse
    (optional, fp32 [tokens, q_heads]) gets the logarithm of every row's softmax sum."""

    def __init__(self, q, cache, page_table, q_start, context, out, max_new, max_context, scale=None, window=0,
                 sinks=0, lse=None, status=None, workspace=None):
        _check(q, "q", dtype=str(cache.k.dtype))
        if q.dim() != 3 or q.shape[2] != cache.head_dim or q.shape[1] % cache.kv_heads:
            raise ValueError(f"q has shape {tuple(q.shape)}: [tokens, q_heads, head_dim] over {cache.kv_heads} KV heads "
                             f"of {cache.head_dim} expected")
        _check(out, "out", q.shape, str(q.dtype))
        _check(lse, "lse", q.shape[:2], "torch.float32", optional=True)
        if lse is not None and not lse.is_contiguous():
            raise ValueError("lse is not contiguous")
        _check_sequences(page_table, q_start, context, status)
        if not all(0 <= x < 1 << 30 for x in (window, sinks, max_new, max_context)):
            raise ValueError("window, sinks, max_new and max_context lie in [0, 2^30)")
        block = _native.Attention(
            q=_ptr(q), out=_ptr(out), lse=_ptr(lse), k_pages=_ptr(cache.k), v_pages=_ptr(cache.v),
            page_table=_ptr(page_table), q_start=_ptr(q_start), context=_ptr(context), status=_ptr(status),
            q_token_stride=_stride(q, 0), q_head_stride=_stride(q, 1), out_token_stride=_stride(out, 0),
            out_head_stride=_stride(out, 1), k_page_stride=_stride(cache.k, 0), k_head_stride=_stride(cache.k, 1),
            k_slot_stride=_stride(cache.k, 2), v_page_stride=_stride(cache.v, 0), v_head_stride=_stride(cache.v, 1),
            v_slot_stride=_stride(cache.v, 2), table_stride=_stride(page_table, 0), tokens=q.shape[0],
            sequences=page_table.shape[0], q_heads=q.shape[1], kv_heads=cache.kv_heads, head_dim=cache.head_dim,
            pages=cache.pages, page_size=cache.page_size, table_width=page_table.shape[1],
            max_new=min(int(max_new), q.shape[0]), max_context=int(max_context), window=int(window), sinks=int(sinks),
            dtype=_dtype(q, "q"), scale=cache.head_dim ** -0.5 if scale is None else float(scale))
        self._bind("attention", block, (q, out, lse, cache.k, cache.v, page_table, q_start, context, status), workspace)


class AppendKV(_Call):
    """Rotary positions of q and k, and k and v into their slots of `cache`. q [tokens, q_heads, head_dim] and
    q_out may be None (keys and values alone); cos and sin are fp32 [positions, rot / 2], or None for no
    rotation."""

    def __init__(self, q, k, v, cos, sin, cache, page_table, q_start, context, q_out, interleaved=False, status=None):
        dtype = str(cache.k.dtype)
        _check(k, "k", dtype=dtype)
        if k.dim() != 3 or tuple(k.shape[1:]) != (cache.kv_heads, cache.head_dim):
            raise ValueError(f"k has shape {tuple(k.shape)}: [tokens, {cache.kv_heads}, {cache.head_dim}] expected")
        _check(v, "v", k.shape, dtype)
        q_heads = 0
        if q is not None:
            _check(q, "q", dtype=dtype)
            if q.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != cache.head_dim:
                raise ValueError(f"q has shape {tuple(q.shape)}: [{k.shape[0]}, q_heads, {cache.head_dim}] expected")
            _check(q_out, "q_out", q.shape, dtype)
            q_heads = q.shape[1]
        _check(cos, "cos", dtype="torch.float32", optional=True)
        rot = positions = 0
        if cos is not None:
            if cos.dim() != 2 or not cos.is_contiguous():
                raise ValueError("cos and sin are contiguous [positions, rot / 2]")
            _check(sin, "sin", cos.shape, "torch.float32")
            if not sin.is_contiguous():
                raise ValueError("cos and sin are contiguous [positions, rot / 2]")
            positions, rot = cos.shape[0], 2 * cos.shape[1]
        _check_sequences(page_table, q_start, context, status)
        block = _native.Append(
            q=_ptr(q), k=_ptr(k), v=_ptr(v), cos=_ptr(cos), sin=_ptr(sin) if rot else None,
            q_out=_ptr(q_out) if q_heads else None, k_pages=_ptr(cache.k), v_pages=_ptr(cache.v),
            page_table=_ptr(page_table), q_start=_ptr(q_start), context=_ptr(context), status=_ptr(status),
            q_token_stride=q.stride(0) if q_heads else 0, q_head_stride=q.stride(1) if q_heads else 0,
            k_token_stride=k.stride(0), k_head_stride=k.stride(1), v_token_stride=v.stride(0), v_head_stride=v.stride(1),
            q_out_token_stride=q_out.stride(0) if q_heads else 0, q_out_head_stride=q_out.stride(1) if q_heads else 0,
            k_page_stride=cache.k.stride(0), k_head_page_stride=cache.k.stride(1), k_slot_stride=cache.k.stride(2),
            v_page_stride=cache.v.stride(0), v_head_page_stride=cache.v.stride(1), v_slot_stride=cache.v.stride(2),
            table_stride=page_table.stride(0), tokens=k.shape[0], sequences=page_table.shape[0], q_heads=q_heads,
            kv_heads=cache.kv_heads, head_dim=cache.head_dim, rot=rot, positions=positions, pages=cache.pages,
            page_size=cache.page_size, table_width=page_table.shape[1], interleaved=int(bool(interleaved)),
            dtype=_dtype(k, "k"))
        self._bind("append", block, (k, v, q, cos, sin, q_out, cache.k, cache.v, page_table, q_start, context, status))


class BlockNorm(_Call):
    """hidden = residual_scale * residual + gate * post_norm(block) and normed = pre_norm(hidden), rows of
    width columns. hidden or normed may be None; post_weight None leaves the block as it is, gate None is 1;
    gate is [rows, width] or one row [width]. A norm's factors are weight_offset + weight."""

    def __init__(self, block, residual, hidden, normed, pre_weight=None, post_weight=None, gate=None,
                 residual_scale=1.0, weight_offset=0.0, eps=1e-5):
        _check(block, "block")
        if block.dim() != 2:
            raise ValueError("block has the dimensions [rows, width]")
        dtype, width = str(block.dtype), block.shape[1]
        _check(residual, "residual", block.shape, dtype)
        _check(hidden, "hidden", block.shape, dtype, optional=True)
        _check(normed, "normed", block.shape, dtype, optional=True)
        _check(pre_weight, "pre_weight", (width,), dtype, optional=normed is None)
        _check(post_weight, "post_weight", (width,), dtype, optional=True)
        _check(gate, "gate", block.shape if gate is not None and gate.dim() == 2 else (width,), dtype, optional=True)

        def stride(t):
            return t.stride(0) if t is not None and t.dim() == 2 else 0

        args = _native.BlockNorm(
            block=_ptr(block), residual=_ptr(residual), gate=_ptr(gate), post_weight=_ptr(post_weight),
            pre_weight=_ptr(pre_weight), hidden=_ptr(hidden), normed=_ptr(normed), block_stride=stride(block),
            residual_stride=stride(residual), gate_stride=stride(gate), hidden_stride=stride(hidden),
            normed_stride=stride(normed), rows=block.shape[0], width=width, dtype=_dtype(block, "block"),
            residual_scale=float(residual_scale), weight_offset=float(weight_offset), eps=float(eps))
        self._bind("block_norm", args, (block, residual, hidden, normed, pre_weight, post_weight, gate))


class Sampler(_Call):
    """tokens (int32 [rows]) drawn from logits [rows, vocab] with the numbers `uniform` (fp32 [rows] in
    [0, 1)), after temperature, top-k, top-p and min-p (per row, or None). logprob (optional, fp32 [rows]):
    the logarithm of the chosen token's chance among the kept ones."""

    def __init__(self, logits, uniform, tokens, logprob=None, temperature=None, top_k=None, top_p=None, min_p=None,
                 workspace=None):
        _check(logits, "logits")
        if logits.dim() != 2:
            raise ValueError("logits have the dimensions [rows, vocab]")
        rows = logits.shape[:1]
        _check(uniform, "uniform", rows, "torch.float32")
        _check(tokens, "tokens", rows, "torch.int32")
        for t, name in ((logprob, "logprob"), (temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
            _check(t, name, rows, "torch.float32", optional=True)
        _check(top_k, "top_k", rows, "torch.int32", optional=True)
        block = _native.Sample(
            logits=_ptr(logits), uniform=_ptr(uniform), temperature=_ptr(temperature), top_k=_ptr(top_k),
            top_p=_ptr(top_p), min_p=_ptr(min_p), tokens=_ptr(tokens), logprob=_ptr(logprob),
            row_stride=logits.stride(0), rows=logits.shape[0], vocab=logits.shape[1], dtype=_dtype(logits, "logits"))
        self._bind("sample", block, (logits, uniform, tokens, logprob, temperature, top_k, top_p, min_p), workspace)
