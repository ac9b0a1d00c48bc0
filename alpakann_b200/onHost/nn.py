"""alpaka::nn::onHost::nn -- the attention path and the layers around it
(reference: include/alpaka/nn/onHost/nn/{embedding,rms_norm,attention,rope,
softmax,mlp}.hpp).

Same function names, argument order, defaults and error conditions as the
reference; shape errors raise AnnShapeError (a ValueError), the analogue of
std::invalid_argument. `exec` is accepted and ignored.
"""
import ctypes
import enum
import math
from dataclasses import dataclass

import torch

from .._capi import AnnView, check, lib, ref, view
from .._short import ELSEWHERE as _ELSEWHERE, binding
from ._common import ext, fn, gemm, handle, suffix, trace

BTHD, BHTD = 0, 1


def embeddingLookup(queue, exec, tokenIds, embedding, output):
    """onHost/nn/embedding.hpp:17-36. tokenIds: uint32 (int32 accepted, same bits)."""
    if tokenIds.dtype not in (torch.int32, torch.uint32):
        raise TypeError("embeddingLookup expects uint32 token ids")
    check(fn("embedding_lookup", suffix(embedding, output))(handle(queue), ref(tokenIds), ref(embedding),
                                                            ref(output)))


def rmsNorm(queue, exec, input, weight, output, epsilon):
    """onHost/nn/rms_norm.hpp:17-35."""
    check(fn("rms_norm", suffix(input, weight, output))(handle(queue), ref(input), ref(weight), ref(output),
                                                        float(epsilon)))


def embeddingRmsNorm(queue, exec, tokenIds, embedding, weight, output, epsilon):
    """embeddingLookup (onHost/nn/embedding.hpp:17-36) followed by rmsNorm
    (onHost/nn/rms_norm.hpp:17-35) in one launch, bit for bit their result."""
    if tokenIds.dtype not in (torch.int32, torch.uint32):
        raise TypeError("embeddingLookup expects uint32 token ids")
    check(fn("embedding_rms_norm", suffix(embedding, weight, output))(handle(queue), ref(tokenIds), ref(embedding),
                                                                      ref(weight), ref(output), float(epsilon)))


def qkvProjection(queue, input, Wq, Wk, Wv, Q, K, V):
    """onHost/nn/attention.hpp:38-52 (three GEMMs on cuBLAS, no exec)."""
    sfx = suffix(input, Wq, Wk, Wv, Q, K, V)
    check(fn("qkv_projection", sfx)(handle(queue), ref(input), ref(Wq), ref(Wk), ref(Wv), ref(Q), ref(K), ref(V)))


def outputProjection(queue, input, Wo, output):
    """onHost/nn/attention.hpp:112-116."""
    gemm(queue, input, Wo, output)


def outputProjectionResidual(queue, input, Wo, residual, output):
    """outputProjection (onHost/nn/attention.hpp:112-116) then ops::add of the
    residual, fused: output = residual + input . Wo (residual may be output)."""
    check(fn("output_projection_residual", suffix(input, Wo, residual, output))(
        handle(queue), ref(input), ref(Wo), ref(residual), ref(output)))


def kvCacheAppend(queue, exec, kNew, vNew, kCache, vCache, position, cosTable=None, sinTable=None):
    """New K/V rows (BTHD [B,Tn,Hkv,D]) into BHTD caches [B,Hkv,Tcap,D] at tokens
    [position, position + Tn); with RoPE tables K is rotated on the way (as
    ropeInPlace). For an LBHTD cache pass the layer's sub-view."""
    sfx = suffix(kNew, vNew, kCache, vCache)
    c = ref(cosTable) if cosTable is not None else None
    s = ref(sinTable) if sinTable is not None else None
    check(fn("kv_cache_append", sfx)(handle(queue), ref(kNew), ref(vNew), ref(kCache), ref(vCache), c, s,
                                     int(position)))


def _split_tail(args, n_tensors):
    tensors = args[:n_tensors]
    tail = list(args[n_tensors:])
    layout = int(tail[0]) if len(tail) > 0 else BTHD
    offset = int(tail[1]) if len(tail) > 1 else 0
    return tensors, layout, offset


def rope(queue, exec, *args, layout=None, positionOffset=None):
    """onHost/nn/rope.hpp:49-86.
    rope(queue, exec, in, cosTable, sinTable, out, layout=BTHD, positionOffset=0)
    rope(queue, exec, q, k, cosTable, sinTable, outQ, outK, layout=BTHD, positionOffset=0)"""
    n = sum(1 for a in args if isinstance(a, torch.Tensor))
    tensors, lay, off = _split_tail(args, n)
    lay = lay if layout is None else int(layout)
    off = off if positionOffset is None else int(positionOffset)
    if n == 4:
        x, c, s, out = tensors
        check(fn("rope", suffix(x, c, s, out))(handle(queue), ref(x), ref(c), ref(s), ref(out), lay, off))
    elif n == 6:
        q, k, c, s, oq, ok = tensors
        rope(queue, exec, q, c, s, oq, lay, off)
        rope(queue, exec, k, c, s, ok, lay, off)
    else:
        raise TypeError("rope takes 4 or 6 tensors")


def ropeInPlace(queue, exec, *args, layout=None, positionOffset=None):
    """onHost/nn/rope.hpp:96-135, one launch for q and k together.
    ropeInPlace(queue, exec, tensor, cosTable, sinTable, layout=BTHD, positionOffset=0)
    ropeInPlace(queue, exec, q, k, cosTable, sinTable, layout=BTHD, positionOffset=0)"""
    n = sum(1 for a in args if isinstance(a, torch.Tensor))
    tensors, lay, off = _split_tail(args, n)
    lay = lay if layout is None else int(layout)
    off = off if positionOffset is None else int(positionOffset)
    if n == 3:
        t, c, s = tensors
        check(fn("rope_inplace", suffix(t, c, s))(handle(queue), ref(t), None, ref(c), ref(s), lay, off))
    elif n == 4:
        q, k, c, s = tensors
        check(fn("rope_inplace", suffix(q, k, c, s))(handle(queue), ref(q), ref(k), ref(c), ref(s), lay, off))
    else:
        raise TypeError("ropeInPlace takes 3 or 4 tensors")


def attentionScores(queue, exec, Q, K, scores, queriesPerKvGroup=1, kvLayout=BTHD):
    """onHost/nn/attention.hpp:54-81 (unscaled Q.K^T)."""
    if int(queriesPerKvGroup) == 0:
        raise_shape("attentionScores requires queriesPerKvGroup > 0.")
    trace(f"attentionScores q={ext(Q)} k={ext(K)} scores={ext(scores)} queriesPerKvGroup={int(queriesPerKvGroup)}"
          f" layout={'BTHD' if int(kvLayout) == BTHD else 'BHTD'}")
    check(fn("attention_scores", suffix(Q, K, scores))(handle(queue), ref(Q), ref(K), ref(scores),
                                                      int(queriesPerKvGroup), int(kvLayout)))


def attentionApply(queue, exec, probs, values, out, queriesPerKvGroup=1, kvLayout=BTHD):
    """onHost/nn/attention.hpp:83-110."""
    if int(queriesPerKvGroup) == 0:
        raise_shape("attentionApply requires queriesPerKvGroup > 0.")
    trace(f"attentionApply probs={ext(probs)} values={ext(values)} out={ext(out)}"
          f" queriesPerKvGroup={int(queriesPerKvGroup)} layout={'BTHD' if int(kvLayout) == BTHD else 'BHTD'}")
    check(fn("attention_apply", suffix(probs, values, out))(handle(queue), ref(probs), ref(values), ref(out),
                                                           int(queriesPerKvGroup), int(kvLayout)))


def softmax(queue, exec, input, output, axis):
    """onHost/nn/softmax.hpp:26-40."""
    check(fn("softmax", suffix(input, output))(handle(queue), ref(input), ref(output), int(axis)))


def causalSoftmax(queue, exec, input, output, axis, queryAxis, keyAxis):
    """onHost/nn/softmax.hpp:59-80 (top-left causal mask)."""
    check(fn("causal_softmax", suffix(input, output))(handle(queue), ref(input), ref(output), int(axis),
                                                     int(queryAxis), int(keyAxis)))


def maskedSoftmax(queue, exec, input, mask, output, axis):
    """onHost/nn/softmax.hpp:42-57: softmax along axis of input + mask."""
    check(fn("masked_softmax", suffix(input, mask, output))(handle(queue), ref(input), ref(mask), ref(output),
                                                           int(axis)))


# ---- MLP layers (onHost/nn/mlp.hpp) -----------------------------------------
class Activation(enum.IntEnum):
    """nn::Activation (mlp.hpp:52-58)."""
    none = 0
    relu = 1
    silu = 2
    gelu = 3


@dataclass
class WeightView:
    """mlp.hpp:60-69: a layer weight [in, out]; not copied, not kept alive."""
    view: torch.Tensor


@dataclass
class BiasView:
    """mlp.hpp:71-76: a layer bias [out]."""
    view: torch.Tensor


def _unwrap(t):
    return t.view if isinstance(t, (WeightView, BiasView)) else t


def linear(queue, input, weight, output):
    """mlp.hpp:33-37: output = input . weight (row-major [in, out]), cuBLAS."""
    gemm(queue, input, weight, output)


def linearBias(queue, exec, input, weight, bias, output, activation=Activation.none):
    """mlp.hpp:42-47: output = input . weight + bias, with an optional
    activation fused into the bias pass."""
    check(fn("linear_bias", suffix(input, weight, bias, output))(handle(queue), ref(input), ref(weight), ref(bias),
                                                               int(activation), ref(output)))


def mlpForward(queue, exec, input, weights, biases, *args, workspace=None):
    """mlp.hpp:150-246. mlpForward(queue, exec, input, weights, biases,
    activation, output) or (..., hiddenActivation, lastActivation, output).
    weights / biases: sequences of tensors or WeightView / BiasView."""
    if len(args) == 2:
        hidden, last, output = args[0], args[0], args[1]
    elif len(args) == 3:
        hidden, last, output = args
    else:
        raise TypeError("mlpForward(queue, exec, input, weights, biases, [hidden,] activation, output)")
    ws = [_unwrap(w) for w in weights]
    bs = [_unwrap(b) for b in biases]
    if len(ws) == 0:
        raise_shape("mlpForward: at least one layer is required.")
    if len(ws) != len(bs):
        raise_shape("mlpForward: weights and biases must have the same length.")
    sfx = suffix(input, output, *ws, *bs)
    wv = (AnnView * len(ws))(*[view(w) for w in ws])
    bv = (AnnView * len(bs))(*[view(b) for b in bs])
    wptr = workspace.data_ptr() if workspace is not None else None
    wbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(fn("mlp_forward", sfx)(handle(queue), ref(input), len(ws), wv, bv, int(hidden), int(last), ref(output),
                                 wptr, wbytes))


def mlpForwardWorkspaceBytes(input, weights, biases, output):
    """Bytes of scratch mlpForward needs for these shapes (0 for one layer)."""
    ws = [_unwrap(w) for w in weights]
    bs = [_unwrap(b) for b in biases]
    wv = (AnnView * max(1, len(ws)))(*[view(w) for w in ws])
    bv = (AnnView * max(1, len(bs)))(*[view(b) for b in bs])
    out = ctypes.c_uint64(0)
    check(lib.ann_mlp_forward_workspace_bytes(ref(input), len(ws), wv, bv, ref(output), input.element_size(),
                                              ctypes.byref(out)))
    return out.value


def decodeLatent(queue, exec, latent, weight, output):
    """mlp.hpp:277-282: output = latent . weight (no bias, no activation)."""
    gemm(queue, latent, weight, output)


def mlp(queue, exec, input, Wgate, Wup, Wdown, output, workspace=None):
    """mlp.hpp:307-337: output = swiglu(input . Wgate, input . Wup) . Wdown."""
    sfx = suffix(input, Wgate, Wup, Wdown, output)
    wptr = workspace.data_ptr() if workspace is not None else None
    wbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(fn("mlp", sfx)(handle(queue), ref(input), ref(Wgate), ref(Wup), ref(Wdown), ref(output), wptr, wbytes))


def attentionDecode(queue, exec, Q, K, V, out, scale=None, queriesPerKvGroup=1, kvLayout=BHTD):
    """Fused decode pipeline attentionScores -> ops::scale -> softmax(axis 3)
    -> attentionApply in one kernel (test/unit/nn/attention.cpp:675-734 is
    the reference composition). scale defaults to 1/sqrt(D)."""
    sfx = suffix(Q, K, V, out)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.shape[3])
    check(fn("attention_decode", sfx)(handle(queue), ref(Q), ref(K), ref(V), ref(out), float(scale),
                                      int(queriesPerKvGroup), int(kvLayout)))


def attentionPrefill(queue, exec, Q, K, V, out, scale=None, queriesPerKvGroup=1, kvLayout=BTHD, causal=True):
    """Fused prefill pipeline attentionScores -> ops::scale -> causalSoftmax
    (top-left mask) or softmax -> attentionApply in one kernel
    (test/unit/nn/attention.cpp:591-651 is the reference composition).
    scale defaults to 1/sqrt(D)."""
    sfx = suffix(Q, K, V, out)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.shape[3])
    check(fn("attention_prefill", sfx)(handle(queue), ref(Q), ref(K), ref(V), ref(out), float(scale),
                                       int(queriesPerKvGroup), int(kvLayout), 1 if causal else 0))


def attentionDecodeMirror(queue, exec, Q, K, V, out, outMirror, scale=None, queriesPerKvGroup=1, kvLayout=BHTD):
    """attentionDecode whose results are stored through `outMirror`, the NVLink
    multicast address of out's first element, into every rank's copy of the
    output (include/ann_b200.h, multicast outputs); follow it with the buffer's
    barrier on every rank."""
    sfx = suffix(Q, K, V, out)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.shape[3])
    check(fn("attention_decode_mirror", sfx)(handle(queue), ref(Q), ref(K), ref(V), ref(out),
                                             ctypes.c_void_p(int(outMirror)), float(scale), int(queriesPerKvGroup),
                                             int(kvLayout)))


def attentionPrefillMirror(queue, exec, Q, K, V, out, outMirror, scale=None, queriesPerKvGroup=1, kvLayout=BTHD,
                           causal=True):
    """attentionPrefill with the results stored through the multicast address
    `outMirror` into every rank's copy (see attentionDecodeMirror)."""
    sfx = suffix(Q, K, V, out)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.shape[3])
    check(fn("attention_prefill_mirror", sfx)(handle(queue), ref(Q), ref(K), ref(V), ref(out),
                                              ctypes.c_void_p(int(outMirror)), float(scale), int(queriesPerKvGroup),
                                              int(kvLayout), 1 if causal else 0))


# ---- decode on compressed data -----------------------------------------------
# No reference counterpart: rotary positions with a position per token, the KV
# cache in 8 bits, linear layers with 4-bit weights.
class RotaryPairs(enum.IntEnum):
    """Elements of a head vector that rotary turns together."""
    interleaved = 0  # (2p, 2p + 1), as rope
    halves = 1       # (p, p + P), P = number of frequencies


def _refuse(name, dtypes, tensors):
    """Words why the binding found the call's tensors unfit (their element types,
    or not all on one CUDA device)."""
    dev = None
    for what, t in tensors.items():
        want = dtypes.get(what, torch.float32)
        if t is not None and t.dtype != want and not (want == torch.int32 and t.dtype == torch.uint32):
            raise TypeError(f"{name}: {what} must be {want}, got {t.dtype}")
    for what, t in tensors.items():
        if t is None or t.device == dev:
            continue
        if dev is not None:
            raise ValueError(f"{name}: {what} is on {t.device}, other tensors on {dev}")
        dev = t.device
        if dev.type != "cuda":
            raise ValueError(f"{name} needs CUDA tensors, got {what} on {dev}")
    raise TypeError(f"{name}: a tensor of more than 8 dimensions, or an argument that is no tensor")


def _again(rc, name, entry, dtypes, queue, tensors, *scalars):
    """A call of the binding that is not on the current stream of the current device
    with fitting tensors: words its error, or calls it on `queue` or on the current
    stream of the tensors' device."""
    if rc > 0:
        check(rc)
    values = tensors.values()
    dev = next(iter(values)).get_device()
    if queue is not None:
        if isinstance(queue, torch.cuda.Stream) and queue.device.index != dev and dev >= 0:
            raise ValueError(f"{name}: the stream is on {queue.device}, the tensors on cuda:{dev}")
        queue = handle(queue)
    if dev < 0:
        _refuse(name, dtypes, tensors)
    with torch.cuda.device(dev):
        rc = entry(queue, *values, *scalars)
    if rc < 0:
        _refuse(name, dtypes, tensors)
    check(rc)


def rotaryFrequencies(queue, exec, frequencies, base=10000.0, factor=1.0, trainedLength=0, lowTurns=1.0,
                      highTurns=32.0):
    """frequencies[p] = base^(-p/P) into a float64 vector of P pairs. For contexts
    `factor` times the trained ones: every frequency divided by factor
    (trainedLength 0), or by parts: those that turn more than highTurns times
    over trainedLength tokens are kept, those below lowTurns divided, the ones
    between blended linearly."""
    if frequencies.dtype != torch.float64 or frequencies.device.type != "cuda":
        _refuse("rotaryFrequencies", {"frequencies": torch.float64}, {"frequencies": frequencies})
    with torch.cuda.device(frequencies.device):
        check(lib.ann_rotary_frequencies(handle(queue), ref(frequencies), float(base), float(factor),
                                         float(trainedLength), float(lowTurns), float(highTurns)))


_ROTARY_TYPES = {t: {"q": t, "k": t, "outQ": t, "outK": t, "positions": torch.int32, "frequencies": torch.float64}
                 for t in (torch.float32, torch.float64)}


def rotary(queue, exec, q, k, positions, frequencies, outQ, outK, pairs=RotaryPairs.interleaved, layout=BTHD,
           magnitude=1.0, inverse=False):
    """q and k (k and outK may be None) turned by the angles positions *
    frequencies into outQ and outK, which may be q and k themselves. positions:
    int32 [B,T] or [T]; frequencies: float64, P <= D/2 pairs; elements from 2P
    on are copied. inverse applies the transposed rotation: the gradients of q
    and k from those of outQ and outK."""
    entry = binding.rotary_f64 if q.dtype == torch.float64 else binding.rotary_f32
    rc = _ELSEWHERE if queue is not None else entry(None, q, k, positions, frequencies, outQ, outK, pairs, layout,
                                                    magnitude, inverse)
    if rc:
        if q.dtype not in _ROTARY_TYPES:
            suffix(q)
        _again(rc, "rotary", entry, _ROTARY_TYPES[q.dtype], queue,
               {"q": q, "k": k, "positions": positions, "frequencies": frequencies, "outQ": outQ, "outK": outK},
               pairs, layout, magnitude, inverse)


_CACHE_TYPES = {"kCache": torch.int8, "vCache": torch.int8, "positions": torch.int32, "counts": torch.int32,
                "lengths": torch.int32}


def kvCacheAppendQ8(queue, exec, kNew, vNew, kCache, vCache, kScale, vScale, positions, tokensPerScale, counts=None,
                    kvLayout=BHTD):
    """New K/V rows (float32 BTHD [B,Tn,Hkv,D]) into int8 caches [B,Hkv,Tcap,D]
    at tokens [positions[b], positions[b] + counts[b]) (int32 [B]; counts
    defaults to Tn). kScale, vScale: float32 [B, Hkv, ceil(Tcap /
    tokensPerScale)], one scale per head and block of tokens; a block whose
    scale grows has its earlier tokens rounded anew."""
    rc = _ELSEWHERE if queue is not None else binding.kv_cache_append_q8(
        None, kNew, vNew, kCache, vCache, kScale, vScale, positions, counts, tokensPerScale, kvLayout)
    if rc:
        _again(rc, "kvCacheAppendQ8", binding.kv_cache_append_q8, _CACHE_TYPES, queue,
               {"kNew": kNew, "vNew": vNew, "kCache": kCache, "vCache": vCache, "kScale": kScale, "vScale": vScale,
                "positions": positions, "counts": counts}, tokensPerScale, kvLayout)


def kvCacheReadQ8(queue, exec, kCache, vCache, kScale, vScale, kOut, vOut, tokensPerScale, lengths=None,
                  kvLayout=BHTD):
    """The float32 rows that an 8-bit cache stands for, for the tokens before
    lengths[b] (int32 [B], default all of kOut); rows behind are left as they
    were. Feeds attentionPrefill with a cached prefix."""
    rc = _ELSEWHERE if queue is not None else binding.kv_cache_read_q8(
        None, kCache, vCache, kScale, vScale, kOut, vOut, lengths, tokensPerScale, kvLayout)
    if rc:
        _again(rc, "kvCacheReadQ8", binding.kv_cache_read_q8, _CACHE_TYPES, queue,
               {"kCache": kCache, "vCache": vCache, "kScale": kScale, "vScale": vScale, "kOut": kOut, "vOut": vOut,
                "lengths": lengths}, tokensPerScale, kvLayout)


def attentionDecodeQ8(queue, exec, Q, kCache, vCache, kScale, vScale, out, tokensPerScale, lengths=None, scale=None,
                      queriesPerKvGroup=1, kvLayout=BHTD, causal=True):
    """attentionDecode over an 8-bit cache (kvCacheAppendQ8): Q, out float32
    [B,Tq,Hq,D], the last Tq tokens of sequences of lengths[b] keys (int32 [B],
    default the whole cache). causal: query i sees the keys before
    lengths[b] - Tq + 1 + i; a query that sees none gives zeros. scale defaults
    to 1/sqrt(D)."""
    if scale is None:
        scale = 1.0 / math.sqrt(Q.shape[3])
    rc = _ELSEWHERE if queue is not None else binding.attention_decode_q8(
        None, Q, kCache, vCache, kScale, vScale, lengths, out, scale, queriesPerKvGroup, tokensPerScale, kvLayout, causal)
    if rc:
        _again(rc, "attentionDecodeQ8", binding.attention_decode_q8, _CACHE_TYPES, queue,
               {"Q": Q, "kCache": kCache, "vCache": vCache, "kScale": kScale, "vScale": vScale, "lengths": lengths,
                "out": out}, scale, queriesPerKvGroup, tokensPerScale, kvLayout, causal)


def packWeightQ4(queue, exec, weight, packed, scales, groupSize):
    """A float32 weight [K,N] (row-major [in, out]) in 4 bits: packed int32
    [K/8,N], eight inputs a word, scales float32 [ceil(K/groupSize),N]. Once,
    when the weights are loaded."""
    tensors = {"weight": weight, "packed": packed, "scales": scales}
    if (weight.dtype != torch.float32 or packed.dtype not in (torch.int32, torch.uint32) or
            scales.dtype != torch.float32 or weight.device.type != "cuda" or
            not (weight.device == packed.device == scales.device)):
        _refuse("packWeightQ4", {"packed": torch.int32}, tensors)
    with torch.cuda.device(weight.device):
        check(lib.ann_pack_weight_q4_f32(handle(queue), ref(weight), ref(packed), ref(scales), int(groupSize)))


_LINEAR_TYPES = {"packed": torch.int32}


def linearQ4(queue, exec, input, packed, scales, output, groupSize, bias=None, activation=Activation.none,
             residual=None):
    """output = activation(input . W + bias) + residual with W in 4 bits
    (packWeightQ4): linear, linearBias and outputProjectionResidual for the few
    rows of a decode step. residual may be output."""
    rc = _ELSEWHERE if queue is not None else binding.linear_q4(
        None, input, packed, scales, bias, residual, output, groupSize, activation)
    if rc:
        _again(rc, "linearQ4", binding.linear_q4, _LINEAR_TYPES, queue,
               {"input": input, "packed": packed, "scales": scales, "bias": bias, "residual": residual,
                "output": output}, groupSize, activation)


def raise_shape(msg):
    from .._capi import ANN_EINVAL, AnnShapeError
    raise AnnShapeError(ANN_EINVAL, msg)
