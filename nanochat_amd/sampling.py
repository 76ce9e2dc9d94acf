"""A token a row from logits (csrc/sample.hip): temperature, top-k, top-p (nucleus), min-p and allowed-token masks, from
given uniform numbers. The decoder runtime (decoder.py) chooses its own tokens, with noise of its own; this is for callers
that hold the logits, such as a step made of attention.packed_attention and library products."""
import functools
from collections import OrderedDict

import torch

from .attention import _workspace
from .native import check, device_guard, hip_library, pointer, stream


_WORKSPACES: OrderedDict = OrderedDict()
_COUNT_BYTES = 1 << 16   # a workspace's counts lie within its first 64 KiB


@functools.lru_cache(maxsize=256)
def sample_workspace_bytes(rows: int, vocab: int) -> int:
    """nc_sample_workspace_bytes, kept per shape."""
    return hip_library().nc_sample_workspace_bytes(rows, vocab)


def _per_row(t: torch.Tensor | None, name: str, dtype: torch.dtype, logits: torch.Tensor) -> int | None:
    if t is None:
        return None
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 1 or t.size(0) != logits.size(0) or t.get_device() != logits.get_device() or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{logits.size(0)}] tensor on {logits.device}")
    return pointer(t)


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """logits fp32 or bf16 [rows, vocab] (contiguous rows, any row stride), uniform fp32 [rows] in [0, 1) -> tokens int32
    [rows], -1 where no token is allowed.

    Per row: temperature fp32 [rows] (not above 0: the largest logit, the lowest index among equals); top_k int32 [rows]
    (<= 0: all), top_p fp32 [rows] (>= 1: all) and min_p fp32 [rows] (<= 0: all) are each off when None. mask: int32 (or
    uint32) words [rows, >= ceil(vocab / 32)], token t allowed where bit t % 32 of word t // 32 is set (the words of the
    decoder's masks). Of the allowed tokens whose logit is neither NaN nor -inf, with weights exp((z - max z) /
    temperature): the top_k largest stay (the lower index first among equals), of those the tokens with less than top_p of
    their weight strictly above them, of those the ones of at least min_p times the largest; the token is the first, in
    index order, whose running weight exceeds uniform times what is left. A row's token does not depend on the other rows.
    Calls on different streams may overlap.
    A workspace passed in (at least sample_workspace_bytes) must have been zero-filled before its first use and only used
    by these calls since, one stream at a time. Without one, calls on a stream share a cached workspace; a call that is
    being captured into a graph gets one of the graph's own."""
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must be a device tensor [rows, vocab]")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"logits must be torch.float32 or torch.bfloat16, got {logits.dtype}")
    rows, vocab = logits.shape
    if vocab < 1 or vocab > 2 ** 24 or rows > 2 ** 22:
        raise ValueError(f"logits must be [at most 2^22, 1 to 2^24], got {tuple(logits.shape)}")
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits must have contiguous rows that do not overlap")
    settings = [_per_row(t, name, dtype, logits) for t, name, dtype in (
        (uniform, "uniform", torch.float32), (temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32),
        (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32))]
    if mask is not None:
        if mask.dtype not in (torch.int32, torch.uint32):
            raise TypeError(f"mask must be torch.int32 or torch.uint32 words, got {mask.dtype}")
        if (mask.dim() != 2 or mask.size(0) != rows or mask.size(1) < -(-vocab // 32) or mask.device != logits.device or
                not mask.is_contiguous()):
            raise ValueError(f"mask must be contiguous words [{rows}, {-(-vocab // 32)}] on {logits.device}")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    else:
        _per_row(out, "out", torch.int32, logits)
    if rows == 0:
        return out
    need = sample_workspace_bytes(rows, vocab)
    with device_guard(logits):
        if workspace is None:
            if torch.cuda.is_current_stream_capturing():
                workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)
                workspace[:_COUNT_BYTES].zero_()   # on every replay
            else:
                workspace = _workspace(logits.device, need, _WORKSPACES)
        nbytes = workspace.numel() * workspace.element_size()
        if nbytes < need or not workspace.is_contiguous() or workspace.device != logits.device or workspace.data_ptr() % 16:
            raise ValueError(f"workspace must be a contiguous 16-byte aligned tensor of at least {need} bytes on {logits.device}")
        check(hip_library().nc_sample_tokens(
            pointer(logits), logits.dtype == torch.bfloat16, logits.stride(0) if rows > 1 else vocab, rows, vocab,
            *settings, pointer(mask) if mask is not None else None, mask.size(1) if mask is not None else 0,
            pointer(out), pointer(workspace), nbytes, stream()))
    return out
