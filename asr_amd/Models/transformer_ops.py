"""Differentiable operators of Transformer-style encoder layers on the HIP kernels.

    q, k = qk_norm_rope(q, k, q_weight, k_weight)      # per-head RMS norm and rotary positions
    o = bucket_attention(q, k, v, table)               # softmax attention with a learned bias by distance bucket
    y = gated_feed_forward(x, w_gate, w_up, w_down)    # (act(x Wg^T) * (x Wu^T)) Wd^T

Not in the reference, which has sinusoidal relative positions and a plain Swish block in these places
(Models/Transformer_encoder.py:55-137,191-209); ``ConformerEncoderLayer`` takes them as options.  Tensors are float32,
bfloat16 or float16 on the GPU, all of one type unless said otherwise; anything else raises.  Layouts are (batch, frame,
head, width); a head must be contiguous, the other strides are free (views of one packed projection need no copy).
Calls enqueue on the current stream of the tensors' device and return without synchronising; gradients are computed by
kernels too, without atomics: the same call gives the same bits.  First derivatives in reverse mode only: a second derivative,
a forward-mode tangent and a ``torch.jit`` trace raise.  Calls and their backward passes can be captured into a HIP graph; as with
torch's own operations, no eager graph of the same leaves may be alive then.
"""
import ctypes as C
import functools

import torch

from .. import _lib

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _tensor(who, name, t, dim, like=None, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"asr_amd.{who}: {name} must be a tensor on the GPU; the HIP path has no CPU fallback")
    want = dtype if dtype is not None else like.dtype if like is not None else None
    if want is None and t.dtype not in _DTYPES:
        raise RuntimeError(f"asr_amd.{who}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    if want is not None and t.dtype != want:
        raise RuntimeError(f"asr_amd.{who}: {name} must be {want}, got {t.dtype}")
    if t.dim() != dim:
        raise RuntimeError(f"asr_amd.{who}: {name} must have {dim} dimensions, got {tuple(t.shape)}")
    if like is not None and t.device != like.device:
        raise RuntimeError(f"asr_amd.{who}: {name} is on {t.device}, expected {like.device}")


def _like(first, dim, *others):
    """Whether `first` and `others` are tensors on one GPU, of one type that has kernels, with `dim` dimensions: the checks of
    _tensor in a fifth of their time, for calls that pass them."""
    try:
        if not first.is_cuda or first.dtype not in _DTYPES or first.dim() != dim:
            return False
        for t in others:
            if t.dtype != first.dtype or t.device != first.device or t.dim() != dim:
                return False
        return True
    except AttributeError:
        return False


def _weights(first, dim, *others):
    """The same for float32 parameters on the device of `first`."""
    try:
        for t in others:
            if t.dtype != torch.float32 or t.device != first.device or t.dim() != dim:
                return False
        return True
    except AttributeError:
        return False


def _heads(t):
    """t with contiguous heads: itself, or a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ----------------------------------------------------------------------------------------- norm and rotation --
def qk_norm_rope(q, k, q_weight, k_weight, positions=None, rot_dim=None, base=10000.0, eps=1e-6):
    """Root-mean-square norm of every head of q (B, T, H, D) and k (B, T, Hk, D), times q_weight / k_weight (D, float32),
    then the rotation by position in the same pass: elements p and p + rot_dim / 2 turn by
    position * base ** (-2 p / rot_dim); elements from rot_dim (default D) on only pass the norm.  ``positions``: whole
    numbers (T,) or (B, T) on the GPU, by default 0..T-1; for single new frames of long streams the stream's own (angles
    are reduced in float64).  D even, at most 128.  Returns contiguous (q, k), differentiable in all four tensors."""
    who = "qk_norm_rope"
    if not (_like(q, 4, k) and _weights(q, 1, q_weight, k_weight)):
        _tensor(who, "q", q, 4)
        _tensor(who, "k", k, 4, like=q)
        _tensor(who, "q_weight", q_weight, 1, like=q, dtype=torch.float32)
        _tensor(who, "k_weight", k_weight, 1, like=q, dtype=torch.float32)
    B, T, H, D = q.shape
    if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D or (H == 0) != (k.shape[2] == 0):
        raise RuntimeError(f"asr_amd.{who}: q {tuple(q.shape)} and k {tuple(k.shape)} do not match")
    if q_weight.shape[0] != D or k_weight.shape[0] != D:
        raise RuntimeError(f"asr_amd.{who}: the weights must hold one value for each of a head's {D} elements")
    if D % 2 or not 2 <= D <= 128:
        raise RuntimeError(f"asr_amd.{who}: head width {D}: must be even and in [2, 128]")
    rot = D if rot_dim is None else int(rot_dim)
    if rot % 2 or not 0 <= rot <= D:
        raise RuntimeError(f"asr_amd.{who}: rot_dim {rot}: must be even and in [0, {D}]")
    if not base > 0.0 or not eps >= 0.0:
        raise RuntimeError(f"asr_amd.{who}: base must be positive and eps not negative")
    pos = positions
    if pos is not None:
        if not isinstance(pos, torch.Tensor) or pos.device != q.device or pos.dtype not in (torch.int64, torch.int32):
            raise RuntimeError(f"asr_amd.{who}: positions must be a tensor of whole numbers on {q.device}")
        if tuple(pos.shape) not in ((T,), (B, T)):
            raise RuntimeError(f"asr_amd.{who}: positions must be ({T},) or ({B}, {T}), got {tuple(pos.shape)}")
        if pos.dtype != torch.int64 or (T > 1 and pos.stride(-1) != 1):
            pos = pos.long().contiguous()
    q, k, q_weight, k_weight = _heads(q), _heads(k), q_weight.contiguous(), k_weight.contiguous()
    return _lib.native().rope(q, k, q_weight, k_weight, pos, rot, float(base), float(eps))


# ------------------------------------------------------------------------- attention with a bucketed bias --
MAX_DISTANCE = 1024
MAX_BUCKETS = 256


@functools.lru_cache(maxsize=None)
def bucket_edges(num_buckets, max_distance, causal):
    """The distances at which a direction's buckets number first + 1, first + 2, ... begin.  A direction has n = num_buckets
    buckets (half of them where keys may follow the query); the first n // 2 hold one distance each, the rest cut
    [first, max_distance) in equal steps of the logarithm and the last goes on to infinity: edge i is the least whole x with
    (x / first) ** steps >= (max_distance / first) ** i, found in whole numbers, so that no rounding moves a border."""
    n = num_buckets if causal else num_buckets // 2
    first, steps, got = n // 2, n - n // 2, []
    x = first
    for i in range(1, steps):
        want = max_distance ** i * first ** steps
        lo, hi = x, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** steps * first ** i >= want:
                hi = mid
            else:
                lo = mid + 1
        x = lo
        got.append(x)
    return tuple(got)


@functools.lru_cache(maxsize=None)
def _edges_host(num_buckets, max_distance, causal):
    e = bucket_edges(num_buckets, max_distance, causal)
    return (C.c_int32 * max(1, len(e)))(*e)


def _edges(table, causal, reach):
    """Address of the host's list of edges, which stays for the life of the program."""
    return C.addressof(_edges_host(table.shape[0] if table is not None else 2 if causal else 4, reach, causal))


def _per_utterance(who, name, t, B, q):
    if not isinstance(t, torch.Tensor) or t.device != q.device or t.dtype not in (torch.int32, torch.int64) or t.shape != (B,):
        raise RuntimeError(f"asr_amd.{who}: {name} must be ({B},) whole numbers on {q.device}")
    if t.dtype == torch.int64:                    # beyond 2^30 from the keys nothing changes any more
        t = t.clamp(-2 ** 30, 2 ** 30)
    return t.to(torch.int32).contiguous()


def bucket_attention(q, k, v, table=None, lengths=None, keep=None, offset=None, causal=False, max_distance=128, scale=None):
    """softmax(scale q k^T + table[bucket of each key's distance from the query]) v, differentiable in q, k, v and table.

    q (B, Tq, H, D), k and v (B, Tk, Hk, D) with H a multiple of Hk (query head h reads key head h // (H / Hk)), table
    (num_buckets, H) float32, None for no bias, scale 1 / sqrt(D) by default.  Query i of utterance b stands at position offset[b] + i
    (``offset`` (B,), default zeros) and key j at position j; ``bucket_edges`` says how distances fall into buckets: with
    ``causal`` a query reads only the keys up to its own position and all buckets are for the past, otherwise the second half
    of the buckets is for the keys behind the query.  Keys from ``lengths[b]`` on and keys with ``keep[b, j]`` false are left
    out, whatever they hold (infinities and NaN too); a query that no key is left for gets zeros, and passes no gradient.
    D at most 128, num_buckets at most 256, max_distance at most 1024.  Without gradients, calls with few queries
    (one new frame against a cache, one utterance at a time) split the keys over the GPU.

    Scores, statistics and sums are float32.  Between two products float32 keeps 24 bits of the probabilities and score
    gradients, float16 16 or more; bfloat16 keeps 24 (16 with split keys) for the output, 16 for dq and 8 for dk, dv and for the
    output of a call without gradients whose keys are not split: those errors are up to 1.4 of the last rounding, the others' 1.0.  With
    ``causal``, what a later key of the same 128 queries holds reaches an earlier query only if it is infinite or NaN."""
    who = "bucket_attention"
    if not _like(q, 4, k, v):
        _tensor(who, "q", q, 4)
        _tensor(who, "k", k, 4, like=q)
        _tensor(who, "v", v, 4, like=q)
    B, Tq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D or H == 0 or k.shape[2] == 0 or H % k.shape[2]:
        raise RuntimeError(f"asr_amd.{who}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if not 1 <= D <= 128:
        raise RuntimeError(f"asr_amd.{who}: head width {D}: must be in [1, 128]")
    causal, reach = bool(causal), int(max_distance)
    nb = 2 if causal else 4
    if table is not None:
        _tensor(who, "table", table, 2, like=q, dtype=torch.float32)
        nb, table = table.shape[0], table.contiguous()
        if table.shape[1] != H:
            raise RuntimeError(f"asr_amd.{who}: table must be (buckets, {H}), got {tuple(table.shape)}")
    if not 2 <= nb <= MAX_BUCKETS or (not causal and (nb < 4 or nb % 2)):
        raise RuntimeError(f"asr_amd.{who}: {nb} buckets: 2 to {MAX_BUCKETS}, an even number of at least 4 unless causal")
    if not (nb if causal else nb // 2) // 2 < reach <= MAX_DISTANCE:
        raise RuntimeError(f"asr_amd.{who}: max_distance {reach}: must be beyond the single-distance buckets and at most "
                           f"{MAX_DISTANCE}")
    if lengths is not None:
        lengths = _per_utterance(who, "lengths", lengths, B, q)
    if offset is not None:
        offset = _per_utterance(who, "offset", offset, B, q)
    if keep is not None:
        if (not isinstance(keep, torch.Tensor) or keep.device != q.device or keep.dtype not in (torch.bool, torch.uint8)
                or keep.shape != (B, k.shape[1])):
            raise RuntimeError(f"asr_amd.{who}: keep must be ({B}, {k.shape[1]}) truth values on {q.device}")
        keep = keep.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    q, k, v = _heads(q), _heads(k), _heads(v)
    return _lib.native().attention(q, k, v, table, lengths, keep, offset, _edges(table, causal, reach), causal, scale)


# ---------------------------------------------------------------------------------------- gated feed-forward --
ACTIVATIONS = {"swish": 0, "gelu": 1}


def gated_feed_forward(x, w_gate, w_up, w_down, act="swish"):
    """(act(x w_gate^T) * (x w_up^T)) w_down^T over the last axis of x: w_gate and w_up (f, d), w_down (n, f), no biases; act
    "swish" or "gelu" (the exact one).  All four of one type.  The hidden values are formed in float32 and rounded once for
    the second product, each by itself (to 8 bits for bfloat16, 16 for float16, 24 for float32; never out of range), and so are
    their gradients.  The backward keeps only the inputs and forms the hidden values again.  Up to 64 rows the forward takes a
    form that reads the weights once and keeps the hidden values to 16 bits for both 16-bit types, to 24 for float32."""
    who = "gated_feed_forward"
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise RuntimeError(f"asr_amd.{who}: x must be a tensor of at least one dimension")
    if not _like(x, x.dim()) or not (_like(w_gate, 2, w_up, w_down) and w_gate.dtype == x.dtype and w_gate.device == x.device):
        _tensor(who, "x", x, x.dim())
        for n, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
            _tensor(who, n, w, 2, like=x)
    if w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1] or w_down.shape[1] != w_gate.shape[0]:
        raise RuntimeError(f"asr_amd.{who}: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and "
                           f"w_down {tuple(w_down.shape)} do not match")
    if 0 in w_gate.shape or 0 in w_down.shape:
        raise RuntimeError(f"asr_amd.{who}: empty weights")
    if act not in ACTIVATIONS:
        raise RuntimeError(f"asr_amd.{who}: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    ws = [w.contiguous() for w in (w_gate, w_up, w_down)]
    y = _lib.native().ff(x2, *ws, ACTIVATIONS[act])
    return y.view(*x.shape[:-1], y.shape[-1])
