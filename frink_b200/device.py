"""Device-tensor layer over the C ABI: torch CUDA tensors in, torch CUDA tensors
out, on torch's current stream.  torch is used for device memory and streams
only; every computation is a call into `libfrink_b200.so`."""
import ctypes as C
import threading

import numpy as np
import torch

from . import _lib
from ._lib import check, lib

_contexts = {}
_lock = threading.Lock()


def context(device=None):
    """The process-wide context of `device` (`gpu::shared_device`,
    crates/frink-cuda/src/gpu.rs:172-222): created once, used from any thread."""
    if not torch.cuda.is_available():
        raise _lib.DriverInit("no CUDA device is visible; this backend has no CPU path")
    idx = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    with _lock:
        if idx not in _contexts:
            p = C.c_void_p()
            check(lib().fk_init(idx, C.byref(p)))
            _contexts[idx] = p
        return _contexts[idx]


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _f32(t):
    assert t.is_cuda and t.dtype == torch.float32, "expects a float32 CUDA tensor"
    return t.contiguous()


def _i32(t):
    assert t.is_cuda and t.dtype == torch.int32, "expects an int32 CUDA tensor"
    return t.contiguous()


def counters(reset=False, device=None):
    h, d, n = C.c_uint64(), C.c_uint64(), C.c_uint64()
    check(lib().fk_counters(context(device), C.byref(h), C.byref(d), C.byref(n), int(reset)))
    return {"h2d_bytes": h.value, "d2h_bytes": d.value, "launches": n.value}


def device_error(reset=True, device=None):
    """The word a kernel raises when a bounded wait gave up (0 = none)."""
    code = C.c_int()
    check(lib().fk_device_error(context(device), C.byref(code), int(reset)))
    return code.value


class Weights:
    """Resident quantized weights: `n_mats` equally shaped matrices given as
    their GGUF block bytes (numpy / CPU tensor: uploaded; CUDA tensor: copied
    on the device)."""

    def __init__(self, gguf_bytes, kind, rows, cols, n_mats=1, device=None):
        self.kind, self.rows, self.cols, self.n_mats = int(kind), int(rows), int(cols), int(n_mats)
        self._ctx = context(device)
        self._h = C.c_void_p()
        if isinstance(gguf_bytes, torch.Tensor) and gguf_bytes.is_cuda:
            raw = gguf_bytes.contiguous().view(torch.uint8)
            check(lib().fk_register_weights_dev(self._ctx, _ptr(raw), raw.numel(), self.kind, self.n_mats,
                                                self.rows, self.cols, _stream(), C.byref(self._h)))
            self.gguf_bytes = raw.numel()
        else:
            raw = np.ascontiguousarray(gguf_bytes.numpy() if isinstance(gguf_bytes, torch.Tensor) else gguf_bytes, np.uint8).ravel()
            check(lib().fk_register_weights(self._ctx, raw.ctypes.data_as(C.c_void_p), raw.size, self.kind, self.n_mats,
                                            self.rows, self.cols, C.byref(self._h)))
            self.gguf_bytes = raw.size

    @property
    def handle(self):
        if not self._h:
            raise _lib.Invalid("weights were released")
        return self._h

    def release(self):
        if self._h:
            check(lib().fk_release_weights(self._ctx, self._h))
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


def quantize_q8_1(x):
    """f32 CUDA tensor (numel % 32 == 0) -> uint8 CUDA tensor of 36-byte q8_1 blocks."""
    x = _f32(x)
    y = torch.empty(x.numel() // 32 * 36, dtype=torch.uint8, device=x.device)
    check(lib().fk_quantize_q8_1(context(x.device), _stream(), _ptr(x), x.numel(), _ptr(y)))
    return y


def quantize_q8_1_host(x):
    xd = torch.from_numpy(np.ascontiguousarray(x, np.float32).ravel()).cuda()
    return quantize_q8_1(xd).cpu().numpy()


def gemv(w, x, mat=0, out=None):
    """y[b, r] = W[mat][r] . q8_1(x[b]); x is [cols] or [batch <= 8, cols]."""
    x = _f32(x)
    batch = 1 if x.dim() == 1 else x.shape[0]
    assert x.shape[-1] == w.cols, f"x has {x.shape[-1]} columns, weights have {w.cols}"
    y = out if out is not None else torch.empty((batch, w.rows), dtype=torch.float32, device=x.device)
    check(lib().fk_gemv(w._ctx, _stream(), w.handle, mat, _ptr(x), batch, _ptr(y)))
    return y if x.dim() > 1 or out is not None else y[0]


def gemv_fused(w, x, out=None, mat=0, norm_weight=None, eps=0.0, glu_up=None, glu_act=0, accumulate=False, pair_glu=0, allreduce=None, bias=None):
    """gemv with its elementwise neighbours folded in: reads rmsnorm(x) * norm_weight, or
    act(x) * glu_up (x the gate), and/or adds into `out` instead of overwriting it.
    x (and glu_up) are [batch <= 8, cols] with any row stride that is a multiple of 4.
    pair_glu (1 SiLU, 2 gpt-oss): `w` holds gate and up row-interleaved; the result is
    act(gate) * up, [batch, rows / 2].
    allreduce = (`frink_b200.comm.Comm`, channel): `w` is this rank's column range of a row-split
    matrix and the result is summed over the ranks by the matvec's epilogue.
    bias [rows]: added to the result by the same launch (`fk_gemv_biased`; with a norm and/or accumulate only)."""
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
    batch, ld = x.shape[0], x.stride(0) if x.shape[0] > 1 else max(x.stride(0), w.cols)
    if glu_up is not None:
        assert glu_up.shape == x.shape and glu_up.stride(1) == 1 and (batch == 1 or glu_up.stride(0) == x.stride(0))
    y = out if out is not None else torch.empty((batch, w.rows // 2 if pair_glu else w.rows), dtype=torch.float32, device=x.device)
    if bias is not None:
        assert glu_up is None and not pair_glu and allreduce is None and bias.numel() == w.rows
        check(lib().fk_gemv_biased(w._ctx, _stream(), w.handle, mat, _ptr(x), ld, batch, _ptr(y),
                                   _ptr(_f32(norm_weight)) if norm_weight is not None else None, float(eps), _ptr(_f32(bias)), int(bool(accumulate))))
        return y
    if allreduce is not None:
        comm, (off, n_max) = allreduce
        assert not pair_glu
        check(lib().fk_gemv_fused_allreduce(w._ctx, _stream(), w.handle, mat, _ptr(x), ld, batch, _ptr(y),
                                            _ptr(_f32(norm_weight)) if norm_weight is not None else None, float(eps),
                                            _ptr(glu_up) if glu_up is not None else None, int(glu_act), int(bool(accumulate)),
                                            comm._h, off, n_max, comm.timeout_us))
        return y
    check(lib().fk_gemv_fused(w._ctx, _stream(), w.handle, mat, _ptr(x), ld, batch, _ptr(y),
                              _ptr(_f32(norm_weight)) if norm_weight is not None else None, float(eps),
                              _ptr(glu_up) if glu_up is not None else None, int(glu_act), int(bool(accumulate)),
                              int(pair_glu)))
    return y


def rope_kv(q, k, v, n_heads, n_kv, head_dim, pos, theta, neox, k_cache, v_cache, q_norm=None, k_norm=None, eps=0.0):
    """One launch: (Qwen3: per-head RMSNorm of q and k,) rotate q and k in place (rows at
    pos[0] + r) and append k, v to the caches.  q, k, v may be column slices of one buffer."""
    n = q.shape[0]
    assert k.stride(0) == v.stride(0) or n == 1
    check(lib().fk_rope_kv(context(q.device), _stream(), _ptr(q), _ptr(k), _ptr(v), q.stride(0), k.stride(0), n, n_heads, n_kv, head_dim,
                           _ptr(_i32(pos)), float(theta), int(neox), _ptr(k_cache), _ptr(v_cache),
                           _ptr(_f32(q_norm)) if q_norm is not None else None, _ptr(_f32(k_norm)) if k_norm is not None else None, float(eps),
                           min(k_cache.shape[0], v_cache.shape[0])))


def gemv_multi(w, ids, x, out=None, bias=None):
    """Slot j: matrix ids[j] of `w` times x[j] (or the one shared x) -> out[j]; with bias [n_mats, rows], + bias[ids[j]]."""
    ids, x = _i32(ids), _f32(x)
    k = ids.numel()
    stride = 0 if x.dim() == 1 else x.stride(0)
    y = out if out is not None else torch.empty((k, w.rows), dtype=torch.float32, device=x.device)
    if bias is not None:
        check(lib().fk_gemv_multi_biased(w._ctx, _stream(), w.handle, _ptr(ids), k, _ptr(x), None, stride, 0, _ptr(_f32(bias)), _ptr(y)))
        return y
    check(lib().fk_gemv_multi(w._ctx, _stream(), w.handle, _ptr(ids), k, _ptr(x), stride, _ptr(y)))
    return y


def gemv_multi_glu(w, ids, gate, up, act=0, out=None, n_active=None, bias=None):
    """Slot j: matrix ids[j] of `w` times act(gate[j]) * up[j] -> out[j] (gate, up: [k, cols]); with bias, + bias[ids[j]]."""
    ids, gate, up = _i32(ids), _f32(gate), _f32(up)
    k = ids.numel()
    assert gate.shape == up.shape and gate.dim() == 2 and gate.shape[0] == k
    y = out if out is not None else torch.empty((k, w.rows), dtype=torch.float32, device=gate.device)
    if bias is not None:
        assert n_active is None
        check(lib().fk_gemv_multi_biased(w._ctx, _stream(), w.handle, _ptr(ids), k, _ptr(gate), _ptr(up), gate.stride(0), int(act), _ptr(_f32(bias)), _ptr(y)))
        return y
    check(lib().fk_gemv_multi_glu(w._ctx, _stream(), w.handle, _ptr(ids), k, _ptr(gate), _ptr(up), gate.stride(0), int(act), _ptr(y),
                                  _ptr(_i32(n_active)) if n_active is not None else None))
    return y


def gemv_multi_active(w, ids, x, n_active, out):
    """gemv_multi whose slots >= n_active[0] (a device word) are skipped; `out` keeps its contents there."""
    ids, x = _i32(ids), _f32(x)
    stride = 0 if x.dim() == 1 else x.stride(0)
    check(lib().fk_gemv_multi_active(w._ctx, _stream(), w.handle, _ptr(ids), ids.numel(), _ptr(x), stride, _ptr(out), _ptr(_i32(n_active))))
    return out


def moe_local_slots(ids, w, e0, n_local):
    ids, w = _i32(ids).reshape(-1), _f32(w).reshape(-1)
    k = ids.numel()
    oi = torch.empty(k, dtype=torch.int32, device=ids.device)
    ow = torch.empty(k, dtype=torch.float32, device=ids.device)
    on = torch.empty(1, dtype=torch.int32, device=ids.device)
    check(lib().fk_moe_local_slots(context(ids.device), _stream(), _ptr(ids), _ptr(w), k, e0, n_local, _ptr(oi), _ptr(ow), _ptr(on)))
    return oi, ow, on


def add_bias_(y, bias, ids=None):
    """y [n, cols] += bias [cols], or += bias[ids[r]] row by row (the expert of every slot): gpt-oss's projection biases."""
    y2 = y if y.dim() == 2 else y[None]
    assert y2.is_contiguous() and y2.dtype == torch.float32
    check(lib().fk_add_bias(context(y.device), _stream(), _ptr(y2), _ptr(_f32(bias)), _ptr(_i32(ids)) if ids is not None else None, y2.shape[0], y2.shape[1]))
    return y


def gemv_multi_gate_up(gate, up, ids, x, norm_weight=None, eps=0.0, gate_bias=None, up_bias=None, out=None):
    """gate and up of the chosen experts in one launch: out [2 k, rows], rows j < k = gate[ids[j]] in_j, rows k + j =
    up[ids[j]] in_j (in_j = x[j] or the one shared x; with norm_weight, its RMSNorm), plus the experts' bias rows."""
    ids, x = _i32(ids), _f32(x)
    k = ids.numel()
    stride = 0 if x.dim() == 1 else x.stride(0)
    y = out if out is not None else torch.empty((2 * k, gate.rows), dtype=torch.float32, device=x.device)
    check(lib().fk_gemv_multi_gate_up(gate._ctx, _stream(), gate.handle, up.handle, _ptr(ids), k, _ptr(x), stride,
                                      _ptr(_f32(norm_weight)) if norm_weight is not None else None, float(eps),
                                      _ptr(_f32(gate_bias)) if gate_bias is not None else None,
                                      _ptr(_f32(up_bias)) if up_bias is not None else None, _ptr(y)))
    return y


def moe_layer(layer, x, out=None, accumulate=False, biases=None, norm=None):
    """The routed layer in one call (`fk_moe_layer`): `layer` carries router, router_bias, gate / up / down (stacked
    `Weights`), k, mode, act; x [batch, hidden] or [hidden].  The workspace is kept on the layer object, per batch size.
    biases = (gate_b, up_b, down_b), each [n_experts, rows]: gpt-oss's form (`fk_moe_layer_biased`).
    norm = (weight, eps): x is the un-normalized residual stream (at most 8 rows) and the layer's RMSNorm is folded into
    the router and the gate / up launch (`fk_moe_layer_normed`: four launches)."""
    x2 = _f32(x) if x.dim() == 2 else _f32(x)[None]
    batch = x2.shape[0]
    g = layer.gate
    ws = layer.__dict__.setdefault("_ws", {})
    if batch not in ws:
        need = lib().fk_moe_layer_workspace(g.n_mats, layer.k, g.cols, g.rows, batch)
        ws[batch] = torch.empty(need + 256, dtype=torch.uint8, device=x2.device)
    buf = ws[batch]
    base = (buf.data_ptr() + 255) & ~255
    assert not accumulate or out is not None
    o = out if out is not None else torch.empty((batch, g.cols), dtype=torch.float32, device=x2.device)
    o2 = o if o.dim() == 2 else o[None]
    rb = _ptr(_f32(layer.router_bias)) if layer.router_bias is not None else None
    if norm is not None:
        gb, ub, db = (_f32(t) for t in biases) if biases is not None else (None, None, None)
        check(lib().fk_moe_layer_normed(g._ctx, _stream(), _ptr(_f32(layer.router)), rb, g.handle, layer.up.handle, layer.down.handle,
                                        _ptr(gb) if gb is not None else None, _ptr(ub) if ub is not None else None,
                                        _ptr(db) if db is not None else None, layer.k, int(layer.mode), int(layer.act),
                                        _ptr(_f32(norm[0])), float(norm[1]), _ptr(x2), batch, _ptr(o2),
                                        int(bool(accumulate)), C.c_void_p(base), buf.numel() - (base - buf.data_ptr())))
        return o if x.dim() == 2 or out is not None else o[0]
    if biases is not None:
        gb, ub, db = (_f32(t) for t in biases)
        assert gb.shape == (g.n_mats, g.rows) and ub.shape == gb.shape and db.shape == (g.n_mats, g.cols)
        check(lib().fk_moe_layer_biased(g._ctx, _stream(), _ptr(_f32(layer.router)), rb, g.handle, layer.up.handle, layer.down.handle,
                                        _ptr(gb), _ptr(ub), _ptr(db), layer.k, int(layer.mode), int(layer.act), _ptr(x2), batch, _ptr(o2),
                                        int(bool(accumulate)), C.c_void_p(base), buf.numel() - (base - buf.data_ptr())))
        return o if x.dim() == 2 or out is not None else o[0]
    check(lib().fk_moe_layer(g._ctx, _stream(), _ptr(_f32(layer.router)), rb,
                             g.handle, layer.up.handle, layer.down.handle, layer.k, int(layer.mode), int(layer.act), _ptr(x2), batch, _ptr(o2),
                             int(bool(accumulate)), C.c_void_p(base), buf.numel() - (base - buf.data_ptr())))
    return o if x.dim() == 2 or out is not None else o[0]


def moe_local_pairs(ids, w, e0, n_local):
    """ids, w [b, k] -> (local expert per slot, source row per slot, slot of each pair, weight of each pair, slot count):
    the pairs this rank's experts serve, packed to the front as slots."""
    ids, w = _i32(ids), _f32(w)
    k, pairs = ids.shape[-1], ids.numel()
    oi = torch.empty(pairs, dtype=torch.int32, device=ids.device)
    src, po = torch.empty_like(oi), torch.empty_like(oi)
    ow = torch.empty(pairs, dtype=torch.float32, device=ids.device)
    on = torch.empty(1, dtype=torch.int32, device=ids.device)
    check(lib().fk_moe_local_pairs(context(ids.device), _stream(), _ptr(ids), _ptr(w), pairs, k, e0, n_local, _ptr(oi), _ptr(src), _ptr(po), _ptr(ow),
                                   _ptr(on)))
    return oi, src, po, ow, on


def moe_localize(ids, w, e0, n_local):
    """ids, w [batch, k] -> local ids (n_local where another rank owns the expert) and weights (0 there)."""
    ids, w = _i32(ids), _f32(w)
    oi, ow = torch.empty_like(ids), torch.empty_like(w)
    check(lib().fk_moe_localize(context(ids.device), _stream(), _ptr(ids), _ptr(w), ids.numel(), e0, n_local, _ptr(oi), _ptr(ow)))
    return oi, ow


def gemv_isums(w, x, mat=0):
    x = _f32(x)
    run = 16 if w.kind == 14 else 32
    out = torch.empty((w.rows, w.cols // run), dtype=torch.int32, device=x.device)
    check(lib().fk_gemv_isums(w._ctx, _stream(), w.handle, mat, _ptr(x), _ptr(out)))
    return out


def gemm(w, x, mat=0, out=None):
    """out[t, r] = W[mat][r] . q8_1(x[t]); x is [m, cols]."""
    x = _f32(x)
    assert x.dim() == 2 and x.shape[1] == w.cols
    y = out if out is not None else torch.empty((x.shape[0], w.rows), dtype=torch.float32, device=x.device)
    if w.kind in (13, 30):
        # Q5_K and BF16 have no GEMM kernel (fk_gemm answers UNSUPPORTED): batches of 8 through the matvec, the same integers
        for i in range(0, x.shape[0], 8):
            gemv(w, x[i:i + 8], mat=mat, out=y[i:i + 8])
        return y
    check(lib().fk_gemm(w._ctx, _stream(), w.handle, mat, _ptr(x), x.shape[0], _ptr(y)))
    return y


def gemm_isums(w, x, mat=0):
    """(out, isums): `gemm` plus the exact int32 dot of every run, [m, rows, cols / run]."""
    x = _f32(x)
    run = 16 if w.kind == 14 else 32
    y = torch.empty((x.shape[0], w.rows), dtype=torch.float32, device=x.device)
    isums = torch.empty((x.shape[0], w.rows, w.cols // run), dtype=torch.int32, device=x.device)
    check(lib().fk_gemm_isums(w._ctx, _stream(), w.handle, mat, _ptr(x), x.shape[0], _ptr(y), _ptr(isums)))
    return y, isums


def gemm_plan(w, m, grouped=False):
    """(tile, split) that `gemm` or `gemm_grouped` picks for m rows: tokens a CTA covers, CTAs along the columns."""
    tile, split = C.c_int(), C.c_int()
    check(lib().fk_gemm_plan(w._ctx, w.handle, m, int(grouped), C.byref(tile), C.byref(split)))
    return tile.value, split.value


def gemm_tiled(w, x, tile, split, mat=0, group_off=None, gather=None, pairs=None, isums=False):
    """`gemm` (or, with group_off, `gemm_grouped` over `pairs` rows) with a given plan; isums: (out, the integers of `gemm_isums`)."""
    x = _f32(x)
    m = x.shape[0] if group_off is None else pairs
    y = torch.empty((m, w.rows), dtype=torch.float32, device=x.device)
    s = torch.empty((m, w.rows, w.cols // (16 if w.kind == 14 else 32)), dtype=torch.int32, device=x.device) if isums else None
    check(lib().fk_gemm_tiled(w._ctx, _stream(), w.handle, mat, _ptr(group_off), _ptr(gather), _ptr(x), m, _ptr(y), _ptr(s), tile, split))
    return (y, s) if isums else y


def gemm_q8k(w, x, mat=0, out=None):
    """out[t, r] = W[mat][r] . q8_k(x[t]): the GEMM on frink's CPU activation rule (Q4_K weights)."""
    x = _f32(x)
    assert x.dim() == 2 and x.shape[1] == w.cols
    y = out if out is not None else torch.empty((x.shape[0], w.rows), dtype=torch.float32, device=x.device)
    check(lib().fk_gemm_q8k(w._ctx, _stream(), w.handle, mat, _ptr(x), x.shape[0], _ptr(y)))
    return y


def gemm_q8k_isums(w, x, mat=0):
    """(out, isums): `gemm_q8k` plus the exact integers per super-block, [m, rows, cols / 256, 2]."""
    x = _f32(x)
    y = torch.empty((x.shape[0], w.rows), dtype=torch.float32, device=x.device)
    isums = torch.empty((x.shape[0], w.rows, w.cols // 256, 2), dtype=torch.int32, device=x.device)
    check(lib().fk_gemm_q8k_isums(w._ctx, _stream(), w.handle, mat, _ptr(x), x.shape[0], _ptr(y), _ptr(isums)))
    return y, isums


def gemm_static(w, x, mat=0, out=None):
    """`gemm` through the entry point that allocates nothing on the device: its
    scratch is a fixed block inside the library, so it can be used where device
    allocation is off limits (`out` must then be given: torch allocating the
    result would defeat the point).  Shapes too large for the block raise Invalid."""
    x = _f32(x)
    assert x.dim() == 2 and x.shape[1] == w.cols
    y = out if out is not None else torch.empty((x.shape[0], w.rows), dtype=torch.float32, device=x.device)
    check(lib().fk_gemm_static(w._ctx, _stream(), w.handle, mat, _ptr(x), x.shape[0], _ptr(y)))
    return y


def gemm_grouped(w, group_off, gather, x, pairs, out=None):
    """Permuted row p (expert e where group_off[e] <= p < group_off[e+1]) reads
    x[gather[p]] and writes out[p]."""
    x, group_off = _f32(x), _i32(group_off)
    gather = _i32(gather) if gather is not None else None
    y = out if out is not None else torch.empty((pairs, w.rows), dtype=torch.float32, device=x.device)
    check(lib().fk_gemm_grouped(w._ctx, _stream(), w.handle, _ptr(group_off), _ptr(gather), _ptr(x), pairs, _ptr(y)))
    return y


def router_logits(router, x):
    router, x = _f32(router), _f32(x)
    x2 = x if x.dim() == 2 else x[None]
    out = torch.empty((x2.shape[0], router.shape[0]), dtype=torch.float32, device=x.device)
    check(lib().fk_router_logits(context(x.device), _stream(), _ptr(router), _ptr(x2), router.shape[0], router.shape[1],
                                 x2.shape[0], _ptr(out)))
    return out


def router_route(router, x, k, mode, bias=None):
    """router_logits followed by moe_route, one launch: (ids [batch, k], weights [batch, k])."""
    router, x = _f32(router), _f32(x)
    x2 = x if x.dim() == 2 else x[None]
    n, e = x2.shape[0], router.shape[0]
    logits = torch.empty((n, e), dtype=torch.float32, device=x.device)
    ids = torch.empty((n, k), dtype=torch.int32, device=x.device)
    w = torch.empty((n, k), dtype=torch.float32, device=x.device)
    b = _f32(bias) if bias is not None else None
    check(lib().fk_router_route(context(x.device), _stream(), _ptr(router), _ptr(x2), e, router.shape[1], n, _ptr(b), k, mode, _ptr(logits),
                                _ptr(ids), _ptr(w)))
    return ids, w


def moe_route(logits, k, mode, bias=None):
    logits = _f32(logits)
    l2 = logits if logits.dim() == 2 else logits[None]
    ids = torch.empty((l2.shape[0], k), dtype=torch.int32, device=logits.device)
    w = torch.empty((l2.shape[0], k), dtype=torch.float32, device=logits.device)
    b = _f32(bias) if bias is not None else None
    check(lib().fk_moe_route(context(logits.device), _stream(), _ptr(l2), _ptr(b), l2.shape[1], k, mode, l2.shape[0],
                             _ptr(ids), _ptr(w)))
    return ids, w


def moe_permute(ids, n_experts):
    ids = _i32(ids)
    pairs, k = ids.numel(), ids.shape[-1]
    dev = ids.device
    group_off = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    gather = torch.empty(pairs, dtype=torch.int32, device=dev)
    pair_of = torch.empty(pairs, dtype=torch.int32, device=dev)
    check(lib().fk_moe_permute(context(dev), _stream(), _ptr(ids), pairs, k, n_experts, _ptr(group_off), _ptr(gather), _ptr(pair_of)))
    return group_off, gather, pair_of


def glu(gate, up, act=0, out=None):
    gate, up = _f32(gate), _f32(up)
    y = out if out is not None else torch.empty_like(gate)
    check(lib().fk_glu(context(gate.device), _stream(), _ptr(gate), _ptr(up), gate.numel(), act, _ptr(y)))
    return y


def moe_combine(y, pair_of, w, batch, k, out=None, accumulate=False):
    """accumulate: add the combined rows into `out` (the residual stream) instead of overwriting it."""
    y, w = _f32(y), _f32(w)
    n = y.shape[-1]
    assert not accumulate or out is not None
    o = out if out is not None else torch.empty((batch, n), dtype=torch.float32, device=y.device)
    fn = lib().fk_moe_combine_add if accumulate else lib().fk_moe_combine
    check(fn(context(y.device), _stream(), _ptr(y), _ptr(_i32(pair_of)) if pair_of is not None else None, _ptr(w), batch, k, n, _ptr(o)))
    return o


# ---- decoder glue -----------------------------------------------------------
def get_rows(w, ids, mat=0, out=None):
    ids = _i32(ids)
    o = out if out is not None else torch.empty((ids.numel(), w.cols), dtype=torch.float32, device=ids.device)
    check(lib().fk_get_rows(w._ctx, _stream(), w.handle, mat, _ptr(ids), ids.numel(), _ptr(o)))
    return o


def rmsnorm(x, weight, eps, residual=None, out=None):
    """out = rmsnorm(x (+ residual)) * weight; with `residual`, x is updated in place to the sum."""
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    x2 = x if x.dim() == 2 else x[None]
    o = out if out is not None else torch.empty_like(x2)
    r = _f32(residual) if residual is not None else None
    check(lib().fk_rmsnorm(context(x.device), _stream(), _ptr(x2), _ptr(r), _ptr(_f32(weight)), x2.shape[0], x2.shape[1], float(eps), _ptr(o)))
    return o if x.dim() == 2 else o[0]


def rope(x, n_heads, head_dim, pos, theta, neox=False):
    """In place; x is [n_rows, n_heads * head_dim], `pos` an int32 device word."""
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    n_rows = 1 if x.dim() == 1 else x.shape[0]
    check(lib().fk_rope(context(x.device), _stream(), _ptr(x), n_rows, n_heads, head_dim, _ptr(_i32(pos)), float(theta), int(neox)))
    return x


def add_(a, b):
    assert a.is_contiguous() and b.is_contiguous()
    check(lib().fk_add(context(a.device), _stream(), _ptr(a), _ptr(_f32(b)), a.numel()))
    return a


def kv_append(cache, src, pos):
    """cache [T, row] rows [*pos, *pos + n) <- src [n, row]."""
    src = _f32(src)
    n = 1 if src.dim() == 1 else src.shape[0]
    check(lib().fk_kv_append(context(cache.device), _stream(), _ptr(cache), _ptr(src), cache.shape[1], n, _ptr(_i32(pos)), cache.shape[0]))


def _sinks(sinks):
    return _ptr(_f32(sinks)) if sinks is not None else None


def attention(q, k_cache, v_cache, n_heads, n_kv, head_dim, pos, scale=None, out=None, window=0, sinks=None):
    """q: [n, n_heads * head_dim] with any row stride that is a multiple of 4 floats (a column
    slice of a merged q/k/v output works), or one row.  window > 0: only the `window` most recent
    keys; sinks [n_heads]: gpt-oss's per-head logit in the softmax's denominator."""
    assert q.is_cuda and q.dtype == torch.float32 and q.stride(-1) == 1
    q2 = q if q.dim() == 2 else q[None]
    o = out if out is not None else torch.empty((q2.shape[0], n_heads * head_dim), dtype=torch.float32, device=q.device)
    sc = float(scale) if scale is not None else head_dim ** -0.5
    ld = q2.stride(0) if q2.shape[0] > 1 else 0
    check(lib().fk_attention(context(q.device), _stream(), _ptr(q2), ld, _ptr(k_cache), _ptr(v_cache), q2.shape[0], n_heads, n_kv, head_dim,
                             _ptr(_i32(pos)), sc, _ptr(o), min(k_cache.shape[0], v_cache.shape[0]), int(window), _sinks(sinks)))
    return o if q.dim() == 2 else o[0]


def attention_rope_kv(q, k_new, v_new, k_cache, v_cache, n_heads, n_kv, head_dim, pos, theta, neox=False, q_norm=None, k_norm=None, eps=0.0,
                      scale=None, out=None, window=0, sinks=None):
    """One decode row: rotate q and the new k at pos[0] (after Qwen3's head norms when given),
    append k and v to the caches and attend over positions 0 ..= pos[0], in one launch.
    q [1, n_heads*head_dim], k_new / v_new [1, n_kv*head_dim] (column slices are fine)."""
    assert q.shape[0] == 1 and q.stride(-1) == 1 and k_new.stride(-1) == 1 and v_new.stride(-1) == 1
    o = out if out is not None else torch.empty((1, n_heads * head_dim), dtype=torch.float32, device=q.device)
    sc = float(scale) if scale is not None else head_dim ** -0.5
    check(lib().fk_attention_rope_kv(context(q.device), _stream(), _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache), n_heads, n_kv,
                                     head_dim, _ptr(_i32(pos)), sc, float(theta), int(neox),
                                     _ptr(_f32(q_norm)) if q_norm is not None else None, _ptr(_f32(k_norm)) if k_norm is not None else None,
                                     float(eps), _ptr(o), min(k_cache.shape[0], v_cache.shape[0]), int(window), _sinks(sinks)))
    return o


def attention_rope_kv_seqs(q, k_new, v_new, k_caches, v_caches, n_heads, n_kv, head_dim, pos, theta, neox=False, q_norm=None, k_norm=None,
                           eps=0.0, scale=None, out=None, window=0, sinks=None):
    """One decode step of independent sequences: row r of q / k_new / v_new (column slices are fine) is sequence r's
    token at position pos[r]; k_caches / v_caches are [n_seqs, T, n_kv*head_dim]."""
    n = q.shape[0]
    assert k_caches.dim() == 3 and k_caches.is_contiguous() and v_caches.is_contiguous() and k_caches.shape == v_caches.shape and k_caches.shape[0] >= n
    assert q.stride(-1) == 1 and k_new.stride(-1) == 1 and v_new.stride(-1) == 1
    assert pos.dtype == torch.int32 and pos.numel() >= n
    o = out if out is not None else torch.empty((n, n_heads * head_dim), dtype=torch.float32, device=q.device)
    sc = float(scale) if scale is not None else head_dim ** -0.5
    check(lib().fk_attention_rope_kv_seqs(context(q.device), _stream(), _ptr(q), q.stride(0), _ptr(k_new), _ptr(v_new), k_new.stride(0), v_new.stride(0),
                                          _ptr(k_caches), _ptr(v_caches), k_caches.stride(0), n, n_heads, n_kv, head_dim, _ptr(pos), sc,
                                          float(theta), int(neox), _ptr(_f32(q_norm)) if q_norm is not None else None,
                                          _ptr(_f32(k_norm)) if k_norm is not None else None, float(eps), _ptr(o), k_caches.shape[1],
                                          int(window), _sinks(sinks)))
    return o


def argmax(x, out=None):
    x = _f32(x)
    x2 = x if x.dim() == 2 else x[None]
    o = out if out is not None else torch.empty(x2.shape[0], dtype=torch.int32, device=x.device)
    check(lib().fk_argmax(context(x.device), _stream(), _ptr(x2), x2.shape[0], x2.shape[1], _ptr(o)))
    return o


def add_int_(p, v):
    check(lib().fk_add_int(context(p.device), _stream(), _ptr(_i32(p)), int(v)))


# ---- paged KV cache -----------------------------------------------------------
_PAGE_KINDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class _CPages(C.Structure):
    """`fk_pages` of the C ABI."""
    _fields_ = [("data_dev", C.c_void_p), ("table_dev", C.c_void_p), ("lens_dev", C.c_void_p), ("refs_dev", C.c_void_p), ("ws_dev", C.c_void_p),
                ("ws_bytes", C.c_size_t), ("kind", C.c_int), ("n_layers", C.c_int), ("n_pages", C.c_int), ("page", C.c_int), ("n_kv", C.c_int),
                ("head_dim", C.c_int), ("n_seqs", C.c_int), ("max_pages", C.c_int)]


class Pages:
    """A KV cache of pages shared by many sequences: data [n_layers, n_pages, 2, n_kv, page, head_dim] (float32, float16 or
    bfloat16; page 16, 32, 64 or 128), table [n_seqs, max_pages] int32 (-1: no page), lens [n_seqs] int32, refs [n_pages]
    int32.  The tensors stay the caller's; the workspace is this object's, and calls on it belong on one stream at a time.
    A cache of some of the pool's sequences (`seq`, or rows of the table) serves every call but `pages_compact`, which moves
    pages and so needs the rows of all."""

    def __init__(self, data, table, lens, refs, _ws=None):
        if data.dim() != 6 or data.shape[2] != 2 or data.dtype not in _PAGE_KINDS:
            raise _lib.Invalid("pages: data is [n_layers, n_pages, 2, n_kv, page, head_dim] of float32, float16 or bfloat16")
        for t in (data, table, lens, refs):
            if not (t.is_cuda and t.device == data.device and t.is_contiguous()):
                raise _lib.Invalid("pages: data, table, lens and refs are contiguous CUDA tensors of one device")
        for t in (table, lens, refs):
            if t.dtype != torch.int32:
                raise _lib.Invalid("pages: table, lens and refs are int32")
        n_layers, n_pages, _, n_kv, page, hd = data.shape
        if table.dim() != 2 or lens.shape != (table.shape[0],) or refs.shape != (n_pages,):
            raise _lib.Invalid("pages: table [n_seqs, max_pages], lens [n_seqs], refs [n_pages]")
        self.data, self.table, self.lens, self.refs = data, table, lens, refs
        self.n_layers, self.n_pages, self.page, self.n_kv, self.head_dim = n_layers, n_pages, page, n_kv, hd
        self.n_seqs, self.max_pages = table.shape
        self._ctx = context(data.device)
        whole = _ws is None                               # a view goes by its cache's workspace
        if whole:
            need = lib().fk_pages_workspace(self._ctx, n_pages)
            _ws = torch.empty(need + 256, dtype=torch.uint8, device=data.device)
            _ws[:8192 + 256].zero_()                      # the arrival counters; what lies behind them is scratch
            torch.cuda.current_stream(data.device).synchronize()    # whatever stream the first call comes on
        self._ws, self._whole = _ws, whole
        base = (_ws.data_ptr() + 255) & ~255
        self._c = _CPages(data.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(), base, _ws.numel() - (base - _ws.data_ptr()),
                          _PAGE_KINDS[data.dtype], n_layers, n_pages, page, n_kv, hd, self.n_seqs, self.max_pages)
        self._p = C.byref(self._c)
        self._dev, self._scale = data.get_device(), hd ** -0.5

    @classmethod
    def alloc(cls, n_layers, n_pages, page, n_kv, head_dim, n_seqs, max_pages, dtype=torch.bfloat16, device="cuda"):
        """An empty cache."""
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros((n_layers, n_pages, 2, n_kv, page, head_dim), dtype=dtype, device=device), torch.full((n_seqs, max_pages), -1, **i32),
                   torch.zeros(n_seqs, **i32), torch.zeros(n_pages, **i32))

    def seq(self, s):
        """Sequence s alone, on the same pages (a prompt's rows)."""
        if not 0 <= s < self.n_seqs:
            raise _lib.Invalid(f"pages: sequence {s} of {self.n_seqs}")
        return Pages(self.data, self.table[s:s + 1], self.lens[s:s + 1], self.refs, _ws=self._ws)


# These calls are a few microseconds of GPU work: the checks read each attribute once, the stream comes as its plain handle.
_F32, _I32 = torch.float32, torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda i: torch.cuda.current_stream(i).cuda_stream


def _n_new(pg, n_new):
    """(device pointer or None, count) of the rows every sequence gets."""
    if isinstance(n_new, torch.Tensor):
        if n_new.dtype != torch.int32 or n_new.get_device() != pg._dev or n_new.shape != (pg.n_seqs,) or not n_new.is_contiguous():
            raise _lib.Invalid(f"pages: n_new is an int32 tensor of {pg.n_seqs} counts on the pages' device")
        return n_new.data_ptr(), 0
    return None, int(n_new)


def _counts(pg, n_new):
    """The optional counts of a call on rows: which of them are real."""
    if n_new is not None and not isinstance(n_new, torch.Tensor):
        raise _lib.Invalid("pages: the rows' counts are a device tensor (the number of rows a sequence follows from q)")
    return None if n_new is None else _n_new(pg, n_new)[0]


def _ints(dev, what, **ts):
    """Contiguous int32 tensors of one length on a device -> that length."""
    n = {t.numel() for t in ts.values()}
    for name, t in ts.items():
        if t.dtype is not _I32 or t.get_device() != dev or dev < 0 or not t.is_contiguous() or len(n) != 1:
            raise _lib.Invalid(f"{what}: {name} is a contiguous int32 CUDA tensor as long as the others")
    return n.pop()


def pages_moves(tokens, live):
    """What a decode step over sequences moves -> (ids, moves), int32: moves (counts for the calls on pages) is 1 where live is not
    0 and the token is not negative; ids are the tokens, 0 in the place of a negative one."""
    dev = tokens.get_device()
    n = _ints(dev, "pages_moves", tokens=tokens, live=live)
    both = tokens.new_empty(2, n)
    check(lib().fk_pages_moves(_contexts.get(dev) or context(tokens.device), _raw_stream(dev), tokens.data_ptr(), live.data_ptr(), n, both.data_ptr(),
                               both.data_ptr() + 4 * n))
    return both[0], both[1]


def _list(ids):
    return (C.c_int * len(ids))(*ids)


def pages_grow(pg, n_new):
    """Every sequence gets the pages for n_new (an int, or int32 [n_seqs] on the device) tokens more than it holds."""
    check(lib().fk_pages_grow(pg._ctx, _raw_stream(pg._dev), pg._p, *_n_new(pg, n_new)))


def pages_advance(pg, n_new):
    """lens += n_new: the step's tokens are in."""
    check(lib().fk_pages_advance(pg._ctx, _raw_stream(pg._dev), pg._p, *_n_new(pg, n_new)))


def pages_fork(pg, src, dst, n=None):
    """Sequence dst[i] (empty) becomes the first n[i] tokens of src[i] (None, or a negative count: all): whole pages are
    shared, the last part of one is copied in every layer.  Lists of at most 64."""
    src, dst = list(src), list(dst)
    if len(src) != len(dst) or (n is not None and len(n) != len(src)):
        raise _lib.Invalid("pages_fork: lists of one length")
    check(lib().fk_pages_fork(pg._ctx, _raw_stream(pg._dev), pg._p, _list(src), _list(dst), _list(list(n)) if n is not None else None, len(src)))


def pages_free(pg, seqs):
    """The listed sequences give their pages back and hold nothing (at most 64 a call)."""
    seqs = list(seqs)
    check(lib().fk_pages_free(pg._ctx, _raw_stream(pg._dev), pg._p, _list(seqs), len(seqs)))


def pages_compact(pg):
    """Moves the pages in use to the front of the pool -> their number (int32 [1] on the device).  pg's table holds every
    sequence of the pool: one that it leaves out would keep the old numbers of pages that have moved."""
    if not pg._whole:
        raise _lib.Invalid("pages_compact: one sequence's view of a cache (the pages of the others would move under them)")
    used = torch.empty(1, dtype=torch.int32, device=pg.data.device)
    check(lib().fk_pages_compact(pg._ctx, _raw_stream(pg._dev), pg._p, used.data_ptr()))
    return used


def _rows_of(pg, t, width, what):
    """t [n_seqs * rows, width], any row stride -> (number of rows, row stride)."""
    at = t.shape
    if t.dtype is not _F32 or t.get_device() != pg._dev or len(at) != 2:
        raise _lib.Invalid(f"{what}: float32 rows of {width} on the pages' device")
    (n, w), (ld, one) = at, t.stride()
    if w != width or one != 1:
        raise _lib.Invalid(f"{what}: float32 rows of {width}, their values side by side")
    if n == 0 or n % pg.n_seqs:
        raise _lib.Invalid(f"{what}: {n} rows for {pg.n_seqs} sequences")
    if ld < width:
        if n > 1:
            raise _lib.Invalid(f"{what}: rows of {width} floats that lie over one another")
        ld = width
    return n, ld


def _out_like(pg, out, q, n, width, what):
    """The result's tensor: a new one beside q, or the caller's."""
    if out is None:
        return q.new_empty(n, width)
    if out.dtype is not _F32 or out.get_device() != pg._dev or out.shape != (n, width) or not out.is_contiguous():
        raise _lib.Invalid(f"{what}: out is a contiguous float32 tensor of q's shape")
    return out


def _vec(pg, t, n, what):
    """An optional contiguous float32 vector of n values on the pages' device -> its address."""
    if t is None:
        return None
    if t.dtype is not _F32 or t.get_device() != pg._dev or t.numel() != n or not t.is_contiguous():
        raise _lib.Invalid(f"{what}: {n} contiguous float32 values on the pages' device")
    return t.data_ptr()


def rope_kv_paged(q, k, v, pg, layer, n_heads, theta, neox=False, n_new=None, q_norm=None, k_norm=None, eps=0.0, out=None):
    """(Qwen3: per-head RMSNorm of q and k,) rotation of q and k and the append of k and v into the pages of `layer`: q, k, v
    are [n_seqs * rows, heads * head_dim] (column slices are fine), row i of sequence s goes to position lens[s] + i; rows from
    n_new[s] on are skipped.  -> the rotated q (`out` may be q itself where its rows are packed); k stays as it is."""
    hd = pg.head_dim
    n, q_ld = _rows_of(pg, q, n_heads * hd, "rope_kv_paged: q")
    nk, k_ld = _rows_of(pg, k, pg.n_kv * hd, "rope_kv_paged: k")
    nv, v_ld = _rows_of(pg, v, pg.n_kv * hd, "rope_kv_paged: v")
    if nk != n or nv != n:
        raise _lib.Invalid("rope_kv_paged: q, k and v have the same number of rows")
    out = _out_like(pg, out, q, n, n_heads * hd, "rope_kv_paged")
    if n == 1:
        q_ld, k_ld, v_ld = n_heads * hd, pg.n_kv * hd, pg.n_kv * hd
    check(lib().fk_rope_kv_paged(pg._ctx, _raw_stream(pg._dev), pg._p, layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_ld, k_ld, v_ld, n // pg.n_seqs,
                                 _counts(pg, n_new), n_heads, theta, neox, _vec(pg, q_norm, hd, "rope_kv_paged: q_norm"),
                                 _vec(pg, k_norm, hd, "rope_kv_paged: k_norm"), eps, out.data_ptr()))
    return out


def attention_paged(q, pg, layer, n_heads, n_new=None, scale=None, window=0, first=0, sinks=None, out=None):
    """Attention over the pages of `layer`: q [n_seqs * rows, n_heads * head_dim] (rotated; any row stride that is a multiple
    of 4), row i of sequence s at position lens[s] + i, its own key and value appended already.  window > 0: the `window` most
    recent keys and the `first` earliest; sinks [n_heads]: a logit per head in the softmax's denominator.  Rows from n_new[s]
    (int32 [n_seqs]) on are left as they were in `out`."""
    width = n_heads * pg.head_dim
    n, ld = _rows_of(pg, q, width, "attention_paged: q")
    out = _out_like(pg, out, q, n, width, "attention_paged")
    check(lib().fk_attention_paged(pg._ctx, _raw_stream(pg._dev), pg._p, layer, q.data_ptr(), ld if n > 1 else width, n // pg.n_seqs,
                                   _counts(pg, n_new), n_heads, pg._scale if scale is None else scale, window, first,
                                   _vec(pg, sinks, n_heads, "attention_paged: sinks"), out.data_ptr()))
    return out


# ---- rules on logits ------------------------------------------------------------
def logit_rules(logits, history=None, penalties=None, bias=None, mask=None, out=None, tokens=None):
    """What a sampler does to logits [n, vocab] (or one row) before it picks, and the greedy pick -> (changed logits, tokens
    int32 [n]).  history [n, h] int32: the tokens that came before (entries outside the vocabulary are empty places); a token
    that occurs c > 0 times has its logit divided (if positive, else multiplied) by repeat, less c * frequency, less presence
    (penalties: float32 [n, 3], or one triple for all rows: numbers of the host, so not while a graph is captured).  bias [vocab]
    or [n, vocab] is added, then logits whose bit in mask (int32 words [words] or [n, words], bit v % 32 of word v / 32) is clear
    become -inf.  tokens: the largest, ties to the lower index; -1 where nothing is left.  One call of this or of `argmax` at a time
    on a device: they share its context's workspace, captured steps too."""
    x = logits if logits.dim() == 2 else logits[None]
    dev = x.get_device()
    if dev < 0 or x.dtype is not _F32 or x.dim() != 2:
        raise _lib.Invalid("logit_rules: float32 CUDA logits [n, vocab]")
    (n, V), (ld, one) = x.shape, x.stride()
    if one != 1 or n == 0 or V == 0:
        raise _lib.Invalid("logit_rules: float32 CUDA logits [n, vocab], a row's values side by side")
    h, hp, pen, bp, b_ld, mp, m_ld = 0, None, None, None, 0, None, 0
    if history is not None:
        hist = history if history.dim() == 2 else history[None]
        at = hist.shape
        if hist.dtype is not _I32 or hist.get_device() != dev or len(at) != 2 or at[0] != n or not hist.is_contiguous():
            raise _lib.Invalid("logit_rules: history is a contiguous int32 tensor [n, h] beside the logits")
        if penalties is None:
            raise _lib.Invalid("logit_rules: a history needs penalties (repeat, frequency, presence)")
        if not isinstance(penalties, torch.Tensor):
            penalties = torch.tensor([[float(v) for v in penalties]], dtype=torch.float32).to(x.device).expand(n, -1)
        pen = penalties if penalties.is_contiguous() else penalties.contiguous()
        if pen.dtype is not _F32 or pen.get_device() != dev or pen.shape != (n, 3):
            raise _lib.Invalid("logit_rules: penalties are float32 [n, 3]: repeat, frequency, presence")
        h = at[1]
        hp = hist.data_ptr() if h else None
    if bias is not None:
        bp, b_ld = _rule_rows(bias, torch.float32, dev, n, V, "bias is float32 [vocab] or [n, vocab]")
    if mask is not None:
        mp, m_ld = _rule_rows(mask, torch.int32, dev, n, (V + 31) // 32, "mask is int32 words [ceil(vocab / 32)] or [n, ...]")
    if out is None:
        o = x.new_empty(n, V)
    else:
        o = out if out.dim() == 2 else out[None]
        if o.shape != (n, V) or o.dtype is not _F32 or o.get_device() != dev or not o.is_contiguous():
            raise _lib.Invalid("logit_rules: out is a contiguous float32 tensor of the logits' shape")
    if tokens is None:
        tokens = x.new_empty(n, dtype=torch.int32)
    elif tokens.shape != (n,) or tokens.dtype is not _I32 or tokens.get_device() != dev or not tokens.is_contiguous():
        raise _lib.Invalid("logit_rules: tokens is a contiguous int32 tensor [n]")
    ctx = _contexts.get(dev) or context(x.device)
    check(lib().fk_logit_rules(ctx, _raw_stream(dev), x.data_ptr(), ld if n > 1 else V, n, V, hp, h,
                               pen.data_ptr() if pen is not None else None, bp, b_ld, mp, m_ld, o.data_ptr(), tokens.data_ptr()))
    return (o if logits.dim() == 2 else o[0]), tokens


def tokens_join(tokens, moves=None, history=None, at=None):
    """A step's tokens int32 [n], in place: -1 where moves [n] (None: all move) is 0.  With a history int32 [n, h] and at int64 [n]
    the others that are not negative join their rows, history[s, at[s] % h] = token, and at counts on.  -> tokens"""
    dev = tokens.get_device()
    n = _ints(dev, "tokens_join", tokens=tokens) if moves is None else _ints(dev, "tokens_join", tokens=tokens, moves=moves)
    h = 0
    if history is not None:
        h = history.shape[-1]
        if history.dtype is not _I32 or history.get_device() != dev or history.shape != (n, h) or h < 1 or not history.is_contiguous():
            raise _lib.Invalid("tokens_join: history is a contiguous int32 tensor [n, h] beside the tokens")
        if at is None or at.dtype is not torch.int64 or at.get_device() != dev or at.shape != (n,) or not at.is_contiguous():
            raise _lib.Invalid("tokens_join: at is a contiguous int64 tensor [n] beside the tokens")
    check(lib().fk_tokens_join(_contexts.get(dev) or context(tokens.device), _raw_stream(dev), tokens.data_ptr(), None if moves is None else moves.data_ptr(), n,
                               None if history is None else history.data_ptr(), h, None if at is None else at.data_ptr()))
    return tokens


def _rule_rows(t, dtype, dev, n, width, what):
    """A row for all, or a row each -> (address, values between rows: 0 = one for all)."""
    if t.dtype != dtype or t.get_device() != dev or t.dim() not in (1, 2) or t.stride(-1) != 1 or t.shape[-1] < width or (t.dim() == 2 and t.shape[0] != n):
        raise _lib.Invalid(f"logit_rules: {what}")
    return t.data_ptr(), 0 if t.dim() == 1 else t.stride(0) if n > 1 else max(t.stride(0), width)
