"""The operators of a step around the cache, as functions on torch tensors:
rotary positions, attention with a sliding window and first tokens that stay
visible, and the choice of the next token.

Like the cache they launch on the current stream of the tensors' device, need
CUDA tensors and the native library (no CPU path), take no part in autograd
and can be captured into CUDA graphs (they use no scratch memory, so graphs
share none).
"""

from __future__ import annotations

import ctypes as C
import math
import operator
from typing import Any, Dict, Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ._lib import RotaryArgs, SampleArgs, WindowArgs, check, lib
from .cache import _DT, _cur_dev, _on, _raw_stream, _stream

_I3 = C.c_int64 * 3
_I2 = C.c_int64 * 2

# Arguments of calls that passed every check and needed no copy of an input, by
# what was checked: shapes, strides, types and settings, never an address or a
# tensor.  A decode step makes the same few calls again and again; from here
# each costs about half its Python time (a copy of the struct with this call's
# pointers filled in).
_PLANS: Dict[tuple, C.Structure] = {}


def _keep(key: tuple, args: C.Structure) -> None:
    if len(_PLANS) >= 1024:
        _PLANS.clear()
    _PLANS[key] = type(args).from_buffer_copy(args)


def _meta(t: Optional[Tensor]) -> Optional[tuple]:
    return None if t is None else (t.dtype, t.shape, t.stride())


def _ready(index: int, *tensors: Optional[Tensor]) -> bool:
    """All on GPU ``index``, which is the current one, and none asks for
    gradients (none can carry a tangent outside of forward-mode levels): nothing
    is left to check but the plan's key."""
    if index < 0 or _cur_dev is None or _raw_stream is None or _cur_dev() != index or forward_ad._current_level >= 0:
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (t.get_device() != index or (grad and t.requires_grad)):
            return False
    return True


def _same_device(what: str, device: torch.device, **tensors: Optional[Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, the others on {device}")


def _cuda(what: str, device: torch.device) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"{what} needs CUDA tensors (no CPU path)")


def _no_grad(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no derivative: call it on tensors without tangents")


def _setting(what: str, x: Any, kind: type) -> Any:
    """A setting as the plain number it is now (None stays): a 0-dim tensor would
    be found again by its identity, whatever it holds by then."""
    if x is None or x.__class__ is kind:
        return x
    if torch.is_tensor(x):
        _no_grad(what, x)
    return int(operator.index(x)) if kind is int else kind(x)


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors without gaps meet in memory, or two of any kind begin
    at one address.  Others with gaps (slices of one projection's output, whose
    rows alternate) are the caller's to keep apart."""
    def span(t: Tensor) -> Tuple[int, int, bool]:
        n = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + n * t.element_size(), n == t.numel()
    if not a.numel() or not b.numel():
        return False
    if a.data_ptr() == b.data_ptr():
        return True
    (a0, a1, whole_a), (b0, b1, whole_b) = span(a), span(b)
    return whole_a and whole_b and a0 < b1 and b0 < a1


# -- rotary positions ------------------------------------------------------------------

# what a dict of rotary settings may hold; a key from elsewhere could ask for other frequencies
_ROPE_KEYS = frozenset((
    "rope_type", "type", "rope_theta", "partial_rotary_factor", "factor", "original_max_position_embeddings",
    "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale",
    "mscale_all_dim"))


def rotary_frequencies(rotary_dim: int, theta: Optional[float] = None, scaling: Optional[Dict[str, Any]] = None,
                       seq_len: Optional[int] = None, device: Union[str, torch.device, None] = None
                       ) -> Tuple[Tensor, float]:
    """``(inv_freq, scale)`` of :func:`apply_rotary`: the angle per position of
    each of the ``rotary_dim / 2`` pairs (float32, computed in 64 bits) and the
    factor on cosine and sine.

    ``scaling`` takes transformers' ``rope_scaling`` dicts.  ``theta`` is the
    dict's ``rope_theta`` where that is given, else 10000; two that differ are
    refused, and so is a key that is not known here, or a
    ``partial_rotary_factor`` other than 1 (the part of a head that is rotated
    is ``rotary_dim``).  By ``rope_type``:

    * ``"default"`` (or None): ``f_i = theta^(-2i/r)``;
    * ``"linear"``: ``f_i / factor``;
    * ``"dynamic"``: theta grows with ``seq_len`` past
      ``original_max_position_embeddings``;
    * ``"llama3"``: waves longer than ``original / low_freq_factor`` positions
      are stretched by ``factor``, those shorter than
      ``original / high_freq_factor`` kept, those between blended;
    * ``"yarn"``: blended over the pair index between ``beta_fast`` and
      ``beta_slow`` turns in the original context; ``scale`` is
      ``attention_factor``, by default ``g(1)`` of ``g(m) = 0.1 m ln(factor) +
      1``, or ``g(mscale) / g(mscale_all_dim)`` where both are given and not 0."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    cfg = {name: v for name, v in (scaling or {}).items() if v is not None or name == "truncate"}
    kind = cfg.get("rope_type", cfg.get("type", "default"))
    unknown = sorted(str(name) for name in cfg if name not in _ROPE_KEYS)
    if unknown:
        raise NotImplementedError(f"rope_type {kind!r} with {', '.join(unknown)} is not supported")
    given = cfg.get("rope_theta")
    if theta is None:
        theta = 10000.0 if given is None else given
    elif given is not None and given != theta:
        raise ValueError(f"theta is {theta}, the dict's rope_theta {given}")
    if not theta > 0 or not math.isfinite(theta):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    if cfg.get("partial_rotary_factor", 1.0) != 1.0:
        raise ValueError(f"partial_rotary_factor {cfg['partial_rotary_factor']}: give the rotated channels as rotary_dim "
                         "and leave it out")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)

    def need(name: str) -> float:
        v = cfg.get(name)
        if v is None or not math.isfinite(v) or v <= 0:
            raise ValueError(f"rope_type {kind!r} needs a positive {name}, got {v!r}")
        return float(v)

    scale = 1.0
    freq = theta ** (-i / rotary_dim)
    if kind == "linear":
        freq = freq / need("factor")
    elif kind == "dynamic":
        factor, original = need("factor"), need("original_max_position_embeddings")
        if rotary_dim <= 2:
            raise ValueError("rope_type 'dynamic' needs a rotary_dim above 2")
        n = max(float(seq_len) if seq_len is not None else original, original)
        base = theta * (factor * n / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        freq = base ** (-i / rotary_dim)
    elif kind == "llama3":
        factor, original = need("factor"), need("original_max_position_embeddings")
        low, high = need("low_freq_factor"), need("high_freq_factor")
        if high <= low:
            raise ValueError(f"high_freq_factor ({high}) must be above low_freq_factor ({low})")
        turns = original * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    elif kind == "yarn":
        factor, original = need("factor"), need("original_max_position_embeddings")
        fast, slow = float(cfg.get("beta_fast") or 32.0), float(cfg.get("beta_slow") or 1.0)
        if fast < slow:
            raise ValueError(f"beta_fast ({fast}) must not be below beta_slow ({slow})")

        def pair_of(turns: float) -> float:  # the pair that makes so many turns in the original context
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = pair_of(fast), pair_of(slow)
        if cfg.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        ramp = ((i / 2 - lo) / (hi - lo if hi != lo else 0.001)).clamp(0.0, 1.0)
        freq = freq * ((1.0 - ramp) + ramp / factor)

        def growth(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        if "attention_factor" in cfg:
            scale = float(cfg["attention_factor"])
        elif cfg.get("mscale") and cfg.get("mscale_all_dim"):
            scale = growth(need("mscale")) / growth(need("mscale_all_dim"))
        else:
            scale = growth(1.0)
    elif kind != "default":
        raise NotImplementedError(f"rope_type {kind!r} is not supported")
    return freq.to(torch.float32).to(device if device is not None else "cpu"), scale


def apply_rotary(query: Tensor, key: Optional[Tensor], positions: Tensor, inv_freq: Tensor, *,
                 interleaved: bool = False, scale: float = 1.0, inverse: bool = False,
                 out: Optional[Tuple[Tensor, Optional[Tensor]]] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """Rotary positions of ``query`` [B, Hq, T, D] and ``key`` [B, Hkv, T, D]
    (or None), any strides; returns the two rotated, laid out like the inputs.

    ``positions`` ([T], [1, T] or [B, T], int64 or int32) times ``inv_freq``
    (float32 [r/2], r <= D) is the angle of a pair of channels, taken in 64
    bits: ``(x[i], x[i + r/2])``, or ``(x[2i], x[2i+1])`` with
    ``interleaved``.  Channels from r on are copied.  ``scale`` multiplies the
    rotated channels; ``inverse`` turns back (and still multiplies by
    ``scale``).  ``out`` gives the outputs' tensors; each may be its own input
    (in place) and must otherwise not overlap any input."""
    if not (interleaved.__class__ is inverse.__class__ is bool and scale.__class__ is float):
        interleaved, inverse = _setting("apply_rotary", interleaved, bool), _setting("apply_rotary", inverse, bool)
        scale = _setting("apply_rotary", scale, float)
    plan_key = None
    if out is None:
        index = query.get_device()
        if _ready(index, query, key, positions, inv_freq):
            plan_key = ("rotary", query.dtype, query.shape, query.stride(), _meta(key), _meta(positions), _meta(inv_freq),
                        interleaved, scale, inverse)
            plan = _PLANS.get(plan_key)
            if plan is not None:
                a = RotaryArgs.from_buffer_copy(plan)
                q_out, k_out = torch.empty_like(query), None
                a.q, a.q_out = query.data_ptr(), q_out.data_ptr()
                if key is not None:
                    k_out = torch.empty_like(key)
                    a.k, a.k_out = key.data_ptr(), k_out.data_ptr()
                a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
                check(lib().skv_rotary(C.byref(a), _raw_stream(index)), "skv_rotary")
                return q_out, k_out
    _same_device("apply_rotary", query.device, key=key, positions=positions, inv_freq=inv_freq)
    _no_grad("apply_rotary", query, key, positions, inv_freq)
    if query.dim() != 4 or (key is not None and key.dim() != 4):
        raise ValueError("apply_rotary: query and key must be [batch, heads, tokens, channels]")
    B, Hq, T, D = query.shape
    if key is not None and (key.shape[0] != B or key.shape[2] != T or key.shape[3] != D):
        raise ValueError(f"apply_rotary: key {tuple(key.shape)} does not match query {tuple(query.shape)}")
    if query.dtype not in _DT or (key is not None and key.dtype != query.dtype):
        raise NotImplementedError("apply_rotary: query and key must share float32, float16 or bfloat16")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("apply_rotary: inv_freq must be a float32 vector")
    r = 2 * inv_freq.shape[0]
    if not 0 < r <= D:
        raise ValueError(f"apply_rotary: inv_freq has {r // 2} pairs, a head {D} channels")
    given = positions
    if positions.dtype != torch.int64:
        if positions.dtype != torch.int32:
            raise ValueError(f"apply_rotary: positions must be int64 or int32, got {positions.dtype}")
        positions = positions.long()
    pshape = positions.shape
    if pshape[-1:] != (T,) or len(pshape) > 2 or (len(pshape) == 2 and pshape[0] not in (1, B)):
        raise ValueError(f"apply_rotary: positions {tuple(pshape)} must be [{T}], [1, {T}] or [{B}, {T}]")
    ps_b = positions.stride(0) if len(pshape) == 2 and pshape[0] == B else 0
    if out is None:
        _cuda("apply_rotary", query.device)
        q_out = torch.empty_like(query)
        k_out = None if key is None else torch.empty_like(key)
    else:
        q_out, k_out = out
        if (k_out is None) != (key is None):
            raise ValueError("apply_rotary: out needs a tensor for each input")
        _no_grad("apply_rotary", q_out, k_out)
        for name, o, x in (("query", q_out, query), ("key", k_out, key)):
            if o is None:
                continue
            if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device:
                raise ValueError(f"apply_rotary: out for {name} must have its shape, type and device")
            for y in (query, key, positions, inv_freq):
                same = y is x and o.data_ptr() == y.data_ptr() and o.stride() == y.stride()
                if y is not None and not same and _overlap(o, y):
                    raise ValueError(f"apply_rotary: out for {name} overlaps an input")
        if k_out is not None and _overlap(q_out, k_out):
            raise ValueError("apply_rotary: the two outputs overlap")
        if any(n > 1 and s == 0 for o in (q_out, k_out) if o is not None for n, s in zip(o.shape, o.stride())):
            raise ValueError("apply_rotary: an expanded tensor cannot be an output")
    _cuda("apply_rotary", query.device)
    if query.numel() == 0 or T == 0:  # nothing but, perhaps, keys without queries
        if key is not None and key.numel():
            raise ValueError("apply_rotary: keys without queries")
        return q_out, k_out
    # unit stride along the channels: other orders go through a copy
    q, k = _unit(query), None if key is None else _unit(key)
    qo, ko = _unit_like(q_out), None if k_out is None else _unit_like(k_out)
    Hkv = 0 if k is None else k.shape[1]
    if Hkv == 0:
        k = None
    if plan_key is not None and not (q is query and (key is None or k is key) and qo is q_out and ko is k_out
                                     and positions is given and inv_freq.is_contiguous()):
        plan_key = None
    inv_freq = inv_freq.contiguous()
    qs, qos = q.stride(), qo.stride()
    ks, kos = (k.stride(), ko.stride()) if k is not None else ((0,) * 4, (0,) * 4)
    a = RotaryArgs(B, T, Hq, Hkv, D, r, interleaved, inverse, _DT[q.dtype], scale, q.data_ptr(),
                   None if k is None else k.data_ptr(), qo.data_ptr(), None if k is None else ko.data_ptr(),
                   _I3(*qs[:3]), _I3(*ks[:3]), _I3(*qos[:3]), _I3(*kos[:3]), positions.data_ptr(),
                   _I2(ps_b, positions.stride(-1)), inv_freq.data_ptr())
    with _on(q.device):
        check(lib().skv_rotary(C.byref(a), _stream(q.device)), "skv_rotary")
    if plan_key is not None:
        _keep(plan_key, a)
    if qo is not q_out:
        q_out.copy_(qo)
    if ko is not k_out:
        k_out.copy_(ko)
    return q_out, k_out


def _unit(x: Tensor) -> Tensor:
    return x if x.stride(-1) == 1 else x.contiguous()


def _unit_like(x: Tensor) -> Tensor:
    return x if x.stride(-1) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


# -- attention with a sliding window and sinks -------------------------------------------

def _vectors(x: Tensor) -> Tensor:
    """``x``, or a copy when its channels are not in a row or its rows not
    16-byte aligned (as the cache copies such keys and values)."""
    es, st = x.element_size(), x.stride()
    if st[3] == 1 and x.data_ptr() % 16 == 0 and not (st[0] * es % 16 or st[1] * es % 16 or st[2] * es % 16):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def sink_window_attention(query: Tensor, key: Tensor, value: Tensor, *, window: Optional[int] = None,
                          sinks: int = 0, scaling: Optional[float] = None, starts: Optional[Tensor] = None,
                          ends: Optional[Tensor] = None, query_slots: Optional[Tensor] = None,
                          out: Optional[Tensor] = None) -> Tensor:
    """Causal attention in which a query sees the last ``window`` tokens (its
    own among them) and its row's first ``sinks`` tokens.

    ``query`` [B, Hq, T, D]; ``key``/``value`` [B, Hkv, S, D] (Hq a multiple of
    Hkv, D 16, 32, 64 or 128); returns [B, T, Hq, D].  T > 1 is a prompt or a
    chunk of one behind a cache, T = 1 a decode step.

    Row b's tokens sit in slots ``starts[b] <= j < ends[b]`` of key and value
    (int32 [B]; default all S slots), its queries in slots ``query_slots[b] +
    i`` (default: they are the row's last T slots, ``ends[b] - T + i``).  A
    query at slot p sees key j when ``starts <= j <= p < ends`` and ``j -
    starts < sinks`` or ``p - j < window`` (``window=None``: every earlier
    token).  So a left-padded prompt gives ``starts``, a right-padded one
    ``ends`` and zero ``query_slots``, a decode step over a preallocated cache
    ``ends``.  A query that sees no key (padding), or only scores of -inf,
    gets zeros, one with a NaN or +inf among its scores NaN; what a query does
    not see never reaches its output, whatever it holds.  Sums are in 32 bits;
    prompts and chunks of 16-bit types may round the weights to their type
    before the product with ``value``."""
    if window.__class__ is not int or sinks.__class__ is not int or scaling is not None:
        window, sinks = _setting("sink_window_attention", window, int), _setting("sink_window_attention", sinks, int)
        scaling = _setting("sink_window_attention", scaling, float)
    plan_key = None
    if out is None:
        index = query.get_device()
        if _ready(index, query, key, value, starts, ends, query_slots):
            qp, kp, vp = query.data_ptr(), key.data_ptr(), value.data_ptr()
            if not (qp | kp | vp) & 15:
                plan_key = ("window", query.dtype, query.shape, query.stride(), _meta(key), _meta(value), _meta(starts),
                            _meta(ends), _meta(query_slots), window, sinks, scaling)
                plan = _PLANS.get(plan_key)
                if plan is not None:
                    a = WindowArgs.from_buffer_copy(plan)
                    out = torch.empty((a.batch, a.q_tokens, a.num_q_heads, a.head_dim), dtype=query.dtype,
                                      device=query.device)
                    a.q, a.k, a.v, a.out = qp, kp, vp, out.data_ptr()
                    if starts is not None:
                        a.starts = starts.data_ptr()
                    if ends is not None:
                        a.ends = ends.data_ptr()
                    if query_slots is not None:
                        a.query_slots = query_slots.data_ptr()
                    check(lib().skv_window_attention(C.byref(a), _raw_stream(index)), "skv_window_attention")
                    return out
    _same_device("sink_window_attention", query.device, key=key, value=value, starts=starts, ends=ends,
                 query_slots=query_slots, out=out)
    _no_grad("sink_window_attention", query, key, value, out)
    if query.dim() != 4 or key.dim() != 4 or key.shape != value.shape:
        raise ValueError("sink_window_attention: query [B, Hq, T, D], key and value [B, Hkv, S, D] of one shape")
    B, Hq, T, D = query.shape
    Hkv, S = key.shape[1], key.shape[2]
    if key.shape[0] != B or key.shape[3] != D or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"sink_window_attention: key {tuple(key.shape)} does not match query {tuple(query.shape)}")
    dt = _DT.get(query.dtype)
    if dt is None or key.dtype != query.dtype or value.dtype != query.dtype:
        raise NotImplementedError("sink_window_attention: query, key and value must share float32, float16 or bfloat16")
    if window is None:
        window = max(S, 1)
    elif window < 1:
        raise ValueError(f"sink_window_attention: window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sink_window_attention: sinks must be at least 0, got {sinks}")
    for name, t in (("starts", starts), ("ends", ends), ("query_slots", query_slots)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous()):
            raise ValueError(f"sink_window_attention: {name} must be a contiguous int32 tensor of shape [{B}]")
    if D not in (16, 32, 64, 128):
        raise NotImplementedError(f"sink_window_attention: head_dim must be 16, 32, 64 or 128, got {D}")
    if out is None:
        _cuda("sink_window_attention", query.device)
        out = torch.empty(B, T, Hq, D, dtype=query.dtype, device=query.device)
    else:
        if out.shape != (B, T, Hq, D) or out.dtype != query.dtype or not out.is_contiguous():
            raise ValueError(f"sink_window_attention: out must be a contiguous {query.dtype} tensor of shape "
                             f"{(B, T, Hq, D)}")
        if any(_overlap(out, x) for x in (query, key, value)):
            raise ValueError("sink_window_attention: out overlaps an input")
        _cuda("sink_window_attention", query.device)
    if out.numel() == 0:
        return out
    if S == 0:
        return out.zero_()
    q, k, v = _vectors(query), _vectors(key), _vectors(value)
    a = WindowArgs(B, T, S, Hq, Hkv, D, dt, min(window, 0x7fffffff), min(sinks, 0x7fffffff),
                   D ** -0.5 if scaling is None else scaling, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                   _I3(*q.stride()[:3]), _I3(*k.stride()[:3]), _I3(*v.stride()[:3]),
                   None if starts is None else starts.data_ptr(), None if ends is None else ends.data_ptr(),
                   None if query_slots is None else query_slots.data_ptr())
    with _on(q.device):
        check(lib().skv_window_attention(C.byref(a), _stream(q.device)), "skv_window_attention")
    if plan_key is not None and q is query and k is key and v is value:
        _keep(plan_key, a)
    return out


# -- the next token ------------------------------------------------------------------------

def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature: Union[float, Tensor] = 1.0,
                  top_k: Union[int, Tensor] = 0, top_p: Union[float, Tensor] = 1.0,
                  min_p: Union[float, Tensor] = 0.0, out: Optional[Tensor] = None) -> Tensor:
    """The next token of each row, int64 [B], from ``logits`` [B, V] and one
    given random number in [0, 1) per row (``uniform``, float32 [B]).

    Weights are ``exp((logit - largest) / temperature)``.  In descending order
    (equal logits by ascending index) ``top_k > 0`` keeps the first k tokens,
    ``top_p < 1`` the fewest first ones of those whose mass reaches top_p of
    theirs, ``min_p`` those of at least min_p times the largest weight.  The
    token is the first, in the vocabulary's order, at which the cumulative
    kept mass exceeds ``uniform`` times the kept mass.  Weights and sums are in
    64 bits (a top-p cut takes weights to 2^-52 of the largest).

    ``temperature`` 0 takes the largest logit (the lowest index of equal
    ones).  NaN logits count as -inf; a row with nothing above -inf gives -1.
    A setting is a number for all rows or a tensor [B] on the logits' device
    (float32; int32 for top_k), whose values are not checked: a temperature at
    or below 0 or NaN is greedy, a top_k at or below 0, a top_p from 1 on and
    a min_p at or below 0 cut nothing, a top_p at or below 0 keeps one token.
    The largest token is always kept.  V is at most 4,194,304."""
    # `tensors` holds each setting that is one for every row, None for a number; it is empty where all are numbers
    settings, tensors = (temperature, top_k, top_p, min_p), ()
    if not (top_k.__class__ is int and temperature.__class__ is top_p.__class__ is min_p.__class__ is float):
        tensors = tuple(s if torch.is_tensor(s) else None for s in settings)
        settings = tuple(s if t is not None else _setting("sample_tokens", s, kind)
                         for s, t, kind in zip(settings, tensors, (float, int, float, float)))
    plan_key = None
    if out is None:
        index = logits.get_device()
        if _ready(index, logits, uniform, *tensors):
            plan_key = ("sample", logits.dtype, logits.shape, logits.stride(), _meta(uniform),
                        settings if not tensors else tuple(s if t is None else _meta(t) for s, t in zip(settings, tensors)))
            plan = _PLANS.get(plan_key)
            if plan is not None:
                a = SampleArgs.from_buffer_copy(plan)
                out = torch.empty((a.batch,), dtype=torch.int64, device=logits.device)
                a.logits, a.uniform, a.tokens = logits.data_ptr(), uniform.data_ptr(), out.data_ptr()
                for name, t in zip(("temperatures", "top_ks", "top_ps", "min_ps"), tensors):
                    if t is not None:
                        setattr(a, name, t.data_ptr())
                check(lib().skv_sample(C.byref(a), _raw_stream(index)), "skv_sample")
                return out
    _same_device("sample_tokens", logits.device, uniform=uniform, out=out)
    _no_grad("sample_tokens", logits, uniform, *tensors)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"sample_tokens: logits must be [rows, vocabulary], got {tuple(logits.shape)}")
    dt = _DT.get(logits.dtype)
    if dt is None:
        raise NotImplementedError(f"sample_tokens: logits of {logits.dtype} are not supported")
    B, V = logits.shape
    if uniform.dtype != torch.float32 or uniform.shape != (B,) or not uniform.is_contiguous():
        raise ValueError(f"sample_tokens: uniform must be a contiguous float32 tensor of shape [{B}]")
    if out is not None and (out.dtype != torch.int64 or out.shape != (B,) or not out.is_contiguous()):
        raise ValueError(f"sample_tokens: out must be a contiguous int64 tensor of shape [{B}]")
    values, arrays = [], []
    for name, s, dtype in zip(("temperature", "top_k", "top_p", "min_p"), settings,
                              (torch.float32, torch.int32, torch.float32, torch.float32)):
        if torch.is_tensor(s):
            if s.device != logits.device or s.dtype != dtype or s.shape != (B,) or not s.is_contiguous():
                raise ValueError(f"sample_tokens: {name} must be a number or a contiguous {dtype} tensor of shape "
                                 f"[{B}] on {logits.device}")
            arrays.append(s.data_ptr())
            values.append(0)
        else:
            arrays.append(None)
            values.append(s)
    if not (arrays[0] is not None or 0.0 <= values[0] < math.inf):
        raise ValueError(f"sample_tokens: temperature must be finite and at least 0, got {temperature}")
    if not (arrays[1] is not None or values[1] >= 0):
        raise ValueError(f"sample_tokens: top_k must be at least 0, got {top_k}")
    if not (arrays[2] is not None or 0.0 < values[2] <= 1.0):
        raise ValueError(f"sample_tokens: top_p must be in (0, 1], got {top_p}")
    if not (arrays[3] is not None or 0.0 <= values[3] <= 1.0):
        raise ValueError(f"sample_tokens: min_p must be in [0, 1], got {min_p}")
    _cuda("sample_tokens", logits.device)
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
    if B == 0:
        return out
    x = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
    a = SampleArgs(B, V, dt, min(values[1], V), values[0], values[2], values[3], 0, x.data_ptr(), x.stride(0),
                   uniform.data_ptr(), arrays[0], arrays[1], arrays[2], arrays[3], out.data_ptr())
    with _on(x.device):
        check(lib().skv_sample(C.byref(a), _stream(x.device)), "skv_sample")
    if plan_key is not None and x is logits:
        _keep(plan_key, a)
    return out
