"""The LM head at decode batches (``w8a8_dense_gemv`` of libw8a8_gfx950.so).

The reference's LM head is a plain 16-bit ``nn.Linear``; at decode it runs as
``F.linear`` of the final-norm rows (``_decode_linear_rows`` /
``_decode_staged_linear``, nanopointllm/llama/lightweight_runner.py:38-43,
96-99, 676-681).  ``dense_gemv`` computes the same product for up to 16 rows
with a hand-written gfx950 kernel that streams the module's own row-major
weight once (binary32 accumulation, one rounding to the output type, a fixed
summation order, so a row's logits do not depend on the other rows of the
batch).  ``DecodeLMHead`` wraps the module: decode batches take the kernel,
larger batches keep the module's own GEMM (``F.linear``), as the reference
does for prefill.

``token_logprobs`` reads the logits once for the log probabilities of given
tokens, the entropy of each row and its most probable tokens: what scores a
prompt, or accepts drafted tokens.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib

MAX_ROWS = 16
MAX_K = 8192


def dense_gemv_supported(x: torch.Tensor, weight: torch.Tensor,
                         bias: torch.Tensor | None = None) -> bool:
    """Whether ``dense_gemv`` takes these operands (else it raises)."""
    if not (x.is_cuda and weight.is_cuda) or x.dtype not in (torch.float16, torch.bfloat16):
        return False
    if weight.dtype != x.dtype or weight.dim() != 2 or weight.stride(-1) != 1:
        return False
    if bias is not None and (bias.dtype != x.dtype or bias.dim() != 1 or not bias.is_contiguous()):
        return False
    k = x.shape[-1]
    rows = x.numel() // k if k else 0
    return (weight.shape[1] == k and 1 <= rows <= MAX_ROWS and 0 < k <= MAX_K and k % 8 == 0
            and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0)


def dense_gemv(x: torch.Tensor, weight: torch.Tensor,
               bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` for at most 16 rows of 16-bit x on the GPU.

    x [..., K] and weight [N, K] (row-major, unit column stride) share a
    16-bit dtype; the result [..., N] has it too.
    """
    device = _lib.require_cuda(x, weight, bias)
    if x.dtype not in (torch.float16, torch.bfloat16) or weight.dtype != x.dtype:
        raise ValueError("dense_gemv takes binary16 or bfloat16 x and weight of one dtype")
    if bias is not None and bias.dtype != x.dtype:
        raise ValueError("bias must have x's dtype")
    if weight.dim() != 2 or weight.stride(-1) != 1:
        raise ValueError("weight must be a row-major [N, K] matrix")
    k = x.shape[-1]
    n = weight.shape[0]
    if weight.shape[1] != k:
        raise ValueError(f"x has {k} columns, weight {weight.shape[1]}")
    rows = x.reshape(-1, k)
    m = rows.shape[0]
    ld = rows.stride(0) if m > 1 else k
    if rows.stride(-1) != 1 or ld < k or ld % 8 or rows.data_ptr() % 16:
        rows = rows.contiguous()
        ld = k
    if m > MAX_ROWS:
        raise ValueError(f"dense_gemv takes at most {MAX_ROWS} rows (got {m}); "
                         "larger batches are a GEMM")
    y = torch.empty(m, n, device=device, dtype=x.dtype)
    if m and n:
        b = bias.contiguous() if bias is not None else None
        _lib.check(_lib.load().w8a8_dense_gemv(
            rows.data_ptr(), ld, weight.data_ptr(),
            weight.stride(0), b.data_ptr() if b is not None else None, y.data_ptr(), n,
            _lib.dtype_code(x.dtype), m, n, k, _lib.stream_handle(device)), "w8a8_dense_gemv")
    return y.view(*x.shape[:-1], n)


class DecodeLMHead(nn.Module):
    """The model's ``lm_head`` with decode batches on ``dense_gemv``.

    Holds the wrapped module (its weight is used in place, not copied).
    GPU tensors only.  Up to 16 rows with supported operands run the kernel;
    larger batches (and shapes outside the kernel's range) take the module's
    own GEMM on the GPU (the reference's ``F.linear``).
    """

    def __init__(self, linear: nn.Linear) -> None:
        super().__init__()
        self.linear = linear

    @property
    def weight(self) -> torch.Tensor:
        return self.linear.weight

    def forward(self, hidden: torch.Tensor) -> torch.Tensor:
        bias = getattr(self.linear, "bias", None)
        _lib.require_cuda(hidden, self.linear.weight, bias)
        if dense_gemv_supported(hidden, self.linear.weight, bias):
            return dense_gemv(hidden, self.linear.weight, bias)
        return F.linear(hidden, self.linear.weight, bias)


MAX_TOP = 64
MAX_VOCAB = 1 << 20
_LOGIT_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


@lru_cache(maxsize=1024)
def _logprobs_workspace(rows: int, vocab: int, top: int, code: int) -> int:
    return int(_lib.load().w8a8_token_logprobs_workspace_bytes(rows, vocab, top, code))


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                  # float32, the tokens' shape
    entropy: torch.Tensor                   # float32 [...], in nats
    top_logprobs: torch.Tensor | None       # float32 [..., top], falling
    top_tokens: torch.Tensor | None         # int64 [..., top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Log probabilities (natural, ``log_softmax``) of given ``tokens`` under
    ``logits [..., vocab]`` (float16, bfloat16 or float32), with the entropy of
    each row and its ``top`` (at most 64) most probable tokens.

    ``tokens`` (int64) has the rows' shape ``[...]``, or ``[..., n]`` for n
    tokens of each row; -1 (a padded place) gives 0, another number outside the
    vocabulary NaN.  Among equal logits the lowest token comes first.  Sums and
    results are binary32; a logit of -inf has probability 0, a row with +inf,
    NaN or nothing above -inf gives NaN.  No autograd.

    Rows of up to 131072 16-bit logits (65536 binary32), in calls of more than 512
    rows half of that, take one kernel; longer ones are cut and joined by a second.
    A row's last bits may differ between the two, and so between calls of up to and
    of more than 512 rows; otherwise they do not depend on the other rows."""
    # A decode step scores its rows eagerly, bounded by the host: each attribute is
    # read once, sizes of workspaces are kept by call.
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        _lib.require_cuda(logits, tokens)    # raises, naming the reason
    code = _LOGIT_CODES.get(logits.dtype)
    axes = logits.dim() - 1
    if code is None or axes < 0:
        raise ValueError("logits must be float16, bfloat16 or float32 [..., vocab]")
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {MAX_VOCAB} tokens")
    given = tokens.shape
    if tokens.dtype != torch.int64 or given[:axes] != shape or len(given) > axes + 1:
        raise ValueError("tokens must be int64 of the rows' shape, or with one more axis")
    if type(top) is not int or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {MAX_TOP} and at most the vocabulary")
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top=top)
    x = logits if axes == 1 else logits.reshape(-1, vocab)
    rows = x.shape[0]
    ld, step = x.stride()
    if step != 1 and vocab > 1 or ld < vocab and rows > 1:
        x, ld = x.contiguous(), vocab
    elif rows == 1:
        ld = vocab
    per = given[-1] if len(given) > axes else 1
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    logprobs = logits.new_empty(given, dtype=torch.float32)
    entropy = logits.new_empty(shape, dtype=torch.float32)
    best = ids = None
    if top:
        best = logits.new_empty((*shape, top), dtype=torch.float32)
        ids = logits.new_empty((*shape, top), dtype=torch.int64)
    if rows == 0:
        return TokenLogprobs(logprobs, entropy, best, ids)
    need = _logprobs_workspace(rows, vocab, top, code)
    ws = logits.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _lib.check(_lib.load().w8a8_token_logprobs(
        x.data_ptr(), ld, code, tokens.data_ptr(), per, per, top, logprobs.data_ptr(),
        entropy.data_ptr(), best.data_ptr() if top else None, ids.data_ptr() if top else None, rows,
        vocab, None if ws is None else ws.data_ptr(), need,
        torch._C._cuda_getCurrentRawStream(index)), "w8a8_token_logprobs")
    return TokenLogprobs(logprobs, entropy, best, ids)
