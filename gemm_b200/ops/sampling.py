"""Sampling ops (csrc/kernels/sampler.cu): greedy arg-max and temperature / top-k / top-p sampling.

Reference: transformer_sample_topk (common/transformer.h:5415-5467) and sample_token
(server/server_llm.c:220-284).  Ties resolve to the lower token id.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _native

_c, _i, _f, _l, _u64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_long, ctypes.c_ulonglong


def _p(t):
    return _c(t.data_ptr()) if t is not None else _c(0)


def argmax(logits: torch.Tensor, idx_offset: int = 0, want_value: bool = False):
    """Row-wise arg-max of ``logits [B, V]`` (f32 or bf16) -> int32 [B] (+ f32 values)."""
    b, v = logits.shape
    if not logits.is_cuda:
        lf = torch.nan_to_num(logits.float(), nan=-3.4e38)
        val, idx = lf.max(dim=-1)
        # torch.max returns the first maximal index on CPU
        idx = (idx + idx_offset).to(torch.int32)
        return (idx, val) if want_value else idx
    out = torch.empty(b, dtype=torch.int32, device=logits.device)
    val = torch.empty(b, dtype=torch.float32, device=logits.device) if want_value else None
    dt = 0 if logits.dtype == torch.float32 else 1
    stream = _c(_native.stream())
    if v >= 16384:
        chunks = max(1, min(64, 1184 // max(1, b)))
        pv = torch.empty(chunks * b, dtype=torch.float32, device=logits.device)
        pi = torch.empty(chunks * b, dtype=torch.int32, device=logits.device)
        rc = _native.cuda().gb_argmax2(_p(logits), _p(out), _p(val), _p(pv), _p(pi), _i(b), _i(v), _l(logits.stride(0)), _i(dt),
                                       _i(idx_offset), _i(chunks), stream)
        _native.check(rc, "gb_argmax2", n=2)
    else:
        rc = _native.cuda().gb_argmax(_p(logits), _p(out), _p(val), _i(b), _i(v), _l(logits.stride(0)), _i(dt), _i(idx_offset), stream)
        _native.check(rc, "gb_argmax")
    return (out, val) if want_value else out


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, seed: int = 0,
           step: int = 0, step_ctr: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Draw one token per row.  ``temperature <= 0`` means greedy.  At most 1024 candidates are kept.  The random numbers are a
    function of ``(seed, step + step_ctr[0], row)``; ``step_ctr`` (int64 [1], on the logits' device) is read by the kernel, so a
    launch captured in a CUDA graph draws from a new step at every replay."""
    if temperature <= 0.0:
        return argmax(logits)
    b, v = logits.shape
    if not logits.is_cuda:
        return sample_ref(logits, temperature, top_k, top_p, seed, step + (int(step_ctr[0]) if step_ctr is not None else 0))
    out = torch.empty(b, dtype=torch.int32, device=logits.device)
    dt = 0 if logits.dtype == torch.float32 else 1
    rc = _native.cuda().gb_sample(_p(logits), _p(out), _i(b), _i(v), _l(logits.stride(0)), _i(dt), _f(temperature), _i(top_k),
                                  _f(top_p), _u64(seed), _u64(step), _p(step_ctr), _c(_native.stream()))
    _native.check(rc, "gb_sample")
    return out


def candidate_set_ref(logits_row: torch.Tensor, temperature: float, top_k: int, top_p: float):
    """Token ids that may be drawn and their probabilities (descending), for tests."""
    v = logits_row.numel()
    kk = min(1024, v) if top_k <= 0 or top_k > 1024 else min(top_k, v)
    vals, idx = torch.sort(logits_row.float(), descending=True, stable=True)
    vals, idx = vals[:kk], idx[:kk]
    p = torch.softmax(vals / max(temperature, 1e-6), dim=-1)
    if top_p < 1.0:
        cum = torch.cumsum(p, 0)
        keep = int((cum >= top_p).nonzero()[0]) + 1 if bool((cum >= top_p).any()) else kk
        p, idx = p[:keep], idx[:keep]
        p = p / p.sum()
    return idx, p


def sample_ref(logits, temperature, top_k, top_p, seed, step):
    g = torch.Generator().manual_seed(seed * 1000003 + step)
    out = []
    for r in range(logits.shape[0]):
        idx, p = candidate_set_ref(logits[r], temperature, top_k, top_p)
        out.append(int(idx[torch.multinomial(p, 1, generator=g)]))
    return torch.tensor(out, dtype=torch.int32)


def uniform_numbers(seed: int, step: int, rows: int = 1) -> torch.Tensor:
    """Numbers in [0, 1) for ``draw``: f32 ``[rows]`` on the host, a function of ``(seed, step, row)``: the generator that ``sample`` uses on the device."""
    m, out = (1 << 64) - 1, []
    for row in range(rows):
        z = (seed + 0x9E3779B97F4A7C15 * (step + 1) + 0xBF58476D1CE4E5B9 * (row + 1)) & m
        z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9 & m
        z = (z ^ z >> 27) * 0x94D049BB133111EB & m
        z ^= z >> 31
        out.append((z >> 40) / 16777216.0)
    return torch.tensor(out, dtype=torch.float32)


def draw(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=None, top_p=None, min_p=None, want_logprob: bool = False):
    """One token per row of ``logits [B, V]`` (f32 or bf16; rows may lie further apart than V) from given numbers ``uniform [B]`` (f32 in [0, 1)): int32 ``[B]``, with
    ``want_logprob`` also the f32 logarithm of the probability it was drawn with.  ``temperature``, ``top_k`` (0: no limit), ``top_p``, ``min_p``: a number, or a
    tensor ``[B]`` with a value for each row (f32; ``top_k`` int32).

    In the order (logit descending, id ascending): the first ``top_k`` ids; of these the ids that have less than ``top_p`` of the probability in front of them (at
    least one); of these the ids with at least ``min_p`` times the largest probability.  The draw is the first id, in id order, at which the kept probability so
    far exceeds ``uniform`` of it all.  ``temperature <= 0``: the lowest id of the largest logit.  NaN counts as -inf; a row without any logit above -inf answers
    id 0 with logarithm -inf.  Probabilities below 2^-45 of the largest count as zero.  On a GPU a row has at most
    1.6 MB of logits."""
    if logits.dim() != 2 or (logits.dtype is not torch.float32 and logits.dtype is not torch.bfloat16) or logits.shape[1] < 1:
        raise ValueError("logits: a tensor [B, V] in f32 or bf16 is needed")
    b, v = logits.shape
    dev = logits.device
    if v > 1 and logits.stride(1) != 1 or (b > 1 and logits.stride(0) < v):
        raise ValueError("logits: a row's values lie one after the other, and rows do not overlap")
    if uniform.dtype != torch.float32 or uniform.shape != (b,) or uniform.device != dev or not uniform.is_contiguous():
        raise ValueError(f"uniform: a contiguous f32 tensor [{b}] beside the logits is needed")
    given = []
    for name, x, dt, none in (("temperature", temperature, torch.float32, 1.0), ("top_k", top_k, torch.int32, 0), ("top_p", top_p, torch.float32, 1.0),
                              ("min_p", min_p, torch.float32, 0.0)):
        if torch.is_tensor(x):
            if x.dtype is not dt or x.shape != (b,) or x.device != dev or not x.is_contiguous():
                raise ValueError(f"{name}: a contiguous {dt} tensor [{b}] beside the logits is needed")
            given.append((x, none))
        else:
            given.append((None, none if x is None else type(none)(x) if x is not top_k else max(-1, min(int(x), 2 ** 31 - 1))))
    if not logits.is_cuda:
        token, logprob = draw_ref(logits, uniform, *(x if x is not None else y for x, y in given))
        return (token, logprob) if want_logprob else token
    (t, t0), (k, k0), (p, p0), (m, m0) = given
    with _native.on_device(dev):
        out = uniform.new_empty(b, dtype=torch.int32)
        logprob = uniform.new_empty(b) if want_logprob else None
        ptr = lambda x: x.data_ptr() if x is not None else None                # noqa: E731
        rc = _native.entry("gb_draw", "pliiipp" + "fpipfpf" + "pppp")(
            logits.data_ptr(), logits.stride(0) if b > 1 else v, 0 if logits.dtype is torch.float32 else 1, b, v, uniform.data_ptr(), ptr(t), t0, ptr(k), k0, ptr(p),
            p0, ptr(m), m0, out.data_ptr(), ptr(logprob), _native.status_ptr(), _native.stream())
        _native.check(rc, "gb_draw", n=1 if b else 0)
    return (out, logprob) if want_logprob else out


def draw_ref(logits, uniform, temperature, top_k, top_p, min_p):
    """``draw`` in 64-bit floats: (tokens, logarithms)."""
    b, v = logits.shape
    col = lambda x: torch.as_tensor(x, device=logits.device).float().double().expand(b)[:, None]       # noqa: E731
    t, k, p, m, u = (col(x) for x in (temperature, top_k, top_p, min_p, uniform))
    x = torch.where(logits.isnan(), float("-inf"), logits.double())
    val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(v, device=logits.device)
    k = torch.where(~(t > 0), 1.0, torch.where(k > 0, k, float(v)))
    d = torch.where(val == val[:, :1], 0.0, val - val[:, :1])
    w = torch.where((rank < k) & (val > float("-inf")), torch.exp(d / torch.where(t > 0, t, 1.0)), 0.0)
    w = torch.where(w > 2.0 ** -45, w, 0.0)
    cum = w.cumsum(-1)
    front = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    keep = (front < p * cum[:, -1:]) | ~(p < 1) | (rank == 0)
    keep &= ~(w < m.clamp_max(1.0))
    w = torch.zeros_like(w).scatter_(1, ids, w * keep)
    cdf = w.cumsum(-1)
    u = torch.where(u > 0, u, 0.0)
    pick = (cdf <= u * cdf[:, -1:]).sum(-1, keepdim=True)
    last = v - 1 - (w.flip(1) > 0).to(torch.int8).argmax(-1, keepdim=True)         # u = 1 and above: the last id that can be drawn
    pick = torch.minimum(pick, last)
    none = cdf[:, -1:] == 0
    pick = torch.where(none, 0, pick)
    lp = torch.where(none, float("-inf"), (w.gather(1, pick) / cdf[:, -1:]).log())
    return pick[:, 0].to(torch.int32), lp[:, 0].float()
