"""Python mirror of the reference's llamd-rocm safe wrappers, over the C ABI.

Names, argument meaning and error behaviour follow
crates/llamd-rocm/src/lib.rs so that tests read like the reference's own
(crates/llamd-testing/tests/grouped_expert.rs, rocm_oracle.rs, planar.rs):

  available(), device_count(), device_info(i)          lib.rs:167-257
  DeviceWeights.upload(w, rows, blocks)                lib.rs:277-308
      .matvec(act)                                     lib.rs:319-375
      .matvec_grouped(act, ids, rows)                  lib.rs:434-511
      .bench_kernel_only(act, iters)                   lib.rs:378-431
  quantize_q8k_on_device(x)                            lib.rs:569-623
  matvec_q6k(w, act, rows)                             lib.rs:914-
plus the pieces of llamd-models / llamd-runtime this backend puts on the
device: route (moe.rs:73-113), MoeLayer (layer.rs:230-260 + the router), and
LmHead (the output matvec + argmax).

Validation happens before any device call; a bad argument raises ValueError
(the Rust wrappers' Error::Shape / Error::Other) and a failing C call raises
HipError. There is no CPU fallback anywhere in this module.
"""
from __future__ import annotations

import ctypes as C
import weakref
from dataclasses import dataclass

import numpy as np

from ._lib import HipError, HipUnavailable, check, check_ptr, lib

QK_K = 256
Q6K_BLOCK_BYTES = 210


def _ptr(a: np.ndarray | None):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


@dataclass
class BlockQ8K:
    """Q8_K activations as arrays: d [nb] f32, qs [nb,256] i8, bsums [nb,16] i16
    (crates/llamd-quant/src/dot.rs:52-62)."""
    d: np.ndarray
    qs: np.ndarray
    bsums: np.ndarray

    @property
    def nblocks(self) -> int:
        return self.d.shape[0]


def device_count() -> int:
    return int(lib().llamd_rocm_device_count())


def available() -> bool:
    try:
        return device_count() > 0
    except (HipUnavailable, OSError):
        return False


@dataclass
class DeviceInfo:
    name: str
    arch: str
    total_mem: int
    compute_units: int
    wave_size: int


def device_info(index: int = 0) -> DeviceInfo:
    name = C.create_string_buffer(256)
    arch = C.create_string_buffer(64)
    mem = C.c_size_t()
    cus = C.c_int()
    wave = C.c_int()
    check(lib().llamd_rocm_device_info(index, name, 256, arch, 64, C.byref(mem), C.byref(cus),
                                       C.byref(wave)), "device_info")
    return DeviceInfo(name.value.decode(), arch.value.decode(), mem.value, cus.value, wave.value)


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


def quantize_q8k_on_device(x) -> BlockQ8K:
    x = _f32(x)
    if x.size % QK_K:
        raise ValueError("Q8_K quantizes whole 256-element blocks")
    nb = x.size // QK_K
    qs = np.empty((nb, QK_K), np.int8)
    d = np.empty(nb, np.float32)
    bs = np.empty((nb, 16), np.int16)
    check(lib().llamd_rocm_quantize_q8k(_ptr(x), nb, _ptr(qs), _ptr(d), _ptr(bs)), "quantize_q8k")
    return BlockQ8K(d, qs, bs)


def swiglu_q8k_on_device(gate, up) -> tuple[np.ndarray, BlockQ8K]:
    """act = silu(gate) * up (CpuBackend::silu/mul) and its Q8_K, fused."""
    g, u = _f32(gate), _f32(up)
    if g.shape != u.shape or g.size % QK_K:
        raise ValueError("gate/up must match and be whole 256-element blocks")
    nb = g.size // QK_K
    act = np.empty(g.size, np.float32)
    qs = np.empty((nb, QK_K), np.int8)
    d = np.empty(nb, np.float32)
    bs = np.empty((nb, 16), np.int16)
    check(lib().llamd_hip_swiglu_q8k(_ptr(g), _ptr(u), nb, _ptr(act), _ptr(qs), _ptr(d), _ptr(bs)),
          "swiglu_q8k")
    return act, BlockQ8K(d, qs, bs)


def _act_arrays(act: BlockQ8K | list[BlockQ8K]):
    if isinstance(act, BlockQ8K):
        return np.ascontiguousarray(act.qs, np.int8), np.ascontiguousarray(act.d, np.float32), 1
    qs = np.ascontiguousarray(np.concatenate([a.qs for a in act]), np.int8)
    d = np.ascontiguousarray(np.concatenate([a.d for a in act]), np.float32)
    return qs, d, len(act)


class DeviceWeights:
    """A Q6_K matrix resident on the device, in the tiled layout.

    Owns its allocation; released exactly once (close() or garbage collection),
    like the Rust handle's Drop (crates/llamd-rocm/src/lib.rs:896-907)."""

    def __init__(self, ptr, rows: int, blocks: int, n_expert: int = 1):
        self._ptr = ptr
        self._rows = rows
        self._blocks = blocks
        self._n_expert = n_expert

    @classmethod
    def upload(cls, w, rows: int, blocks: int) -> "DeviceWeights":
        w = np.ascontiguousarray(np.frombuffer(bytes(w), np.uint8) if isinstance(w, (bytes, bytearray))
                                 else w, dtype=np.uint8)
        if rows <= 0 or blocks <= 0:
            raise ValueError("rows and blocks must be positive")
        need = rows * blocks * Q6K_BLOCK_BYTES
        if w.size < need:
            raise ValueError(f"need {need} bytes for {rows}x{blocks} Q6_K blocks, have {w.size}")
        p = check_ptr(lib().llamd_rocm_upload_q6k(_ptr(w), rows, blocks), "upload_q6k")
        return cls(p, rows, blocks)

    @classmethod
    def upload_experts(cls, w, n_expert: int, rows: int, blocks: int) -> "DeviceWeights":
        w = np.ascontiguousarray(w, dtype=np.uint8)
        need = n_expert * rows * blocks * Q6K_BLOCK_BYTES
        if w.size < need:
            raise ValueError(f"need {need} bytes, have {w.size}")
        p = check_ptr(lib().llamd_rocm_upload_q6k_experts(_ptr(w), n_expert, rows, blocks),
                      "upload_q6k_experts")
        return cls(p, rows, blocks, n_expert)

    @property
    def ptr(self):
        return self._ptr

    def rows(self) -> int:
        return self._rows

    def blocks(self) -> int:
        return self._blocks

    def _check_act(self, act: BlockQ8K):
        if act.nblocks < self._blocks:
            raise ValueError(f"activation has {act.nblocks} blocks, weights need {self._blocks}")

    def matvec(self, act: BlockQ8K) -> np.ndarray:
        self._check_act(act)
        qs, d, _ = _act_arrays(act)
        rows = self._rows
        out = np.empty(rows, np.float32)
        check(lib().llamd_rocm_matvec_q6k_resident(self._ptr, _ptr(qs), _ptr(d), _ptr(out),
                                                   self._blocks, rows), "matvec")
        return out

    def matvec_grouped(self, act: BlockQ8K, ids, rows: int) -> np.ndarray:
        """out[e*rows + r] = row r of expert ids[e] against one shared activation."""
        self._check_act(act)
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        if ids.size == 0 or rows <= 0:
            raise ValueError("no experts / zero rows")
        qs, d, _ = _act_arrays(act)
        out = np.empty(rows * ids.size, np.float32)
        check(lib().llamd_rocm_matvec_grouped(self._ptr, _ptr(ids), _ptr(qs), _ptr(d), _ptr(out),
                                              self._blocks, rows, ids.size), "matvec_grouped")
        return out

    def matvec_grouped_pa(self, acts: list[BlockQ8K], ids, rows: int) -> np.ndarray:
        """Like matvec_grouped, slot e with its own activation acts[e]."""
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        if len(acts) != ids.size or ids.size == 0:
            raise ValueError("one activation per routed expert")
        for a in acts:
            self._check_act(a)
        qs, d, _ = _act_arrays(acts)
        out = np.empty(rows * ids.size, np.float32)
        check(lib().llamd_hip_matvec_grouped_pa(self._ptr, _ptr(ids), _ptr(qs), _ptr(d), _ptr(out),
                                                self._blocks, rows, ids.size), "matvec_grouped_pa")
        return out

    def matvec_batched(self, acts: list[BlockQ8K]) -> np.ndarray:
        """out[s, r] for every activation s; weights read once per 16."""
        for a in acts:
            self._check_act(a)
        qs, d, n = _act_arrays(acts)
        out = np.empty((n, self._rows), np.float32)
        check(lib().llamd_hip_matvec_q6k_batched(self._ptr, _ptr(qs), _ptr(d), _ptr(out),
                                                 self._blocks, self._rows, n), "matvec_batched")
        return out

    def dequantize(self) -> np.ndarray:
        if self._n_expert != 1:
            raise ValueError("dequantize one matrix at a time")
        out = np.empty((self._rows, self._blocks * QK_K), np.float32)
        check(lib().llamd_hip_dequant_q6k(self._ptr, self._rows, self._blocks, _ptr(out)),
              "dequant_q6k")
        return out

    def bench_kernel_only(self, act: BlockQ8K, iters: int) -> float:
        qs, d, _ = _act_arrays(act)
        ms = C.c_float()
        check(lib().llamd_rocm_matvec_bench(self._ptr, _ptr(qs), _ptr(d), self._blocks, self._rows,
                                            iters, C.byref(ms)), "matvec_bench")
        return ms.value

    def close(self):
        if self._ptr:
            lib().llamd_rocm_release(self._ptr)
            self._ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Q8_0Weights:
    """A Q8_0 matrix resident on the device (planar layout)."""

    def __init__(self, w, rows: int, k: int):
        w = np.ascontiguousarray(w, dtype=np.uint8)
        if k % 32 or w.size < rows * k // 32 * 34:
            raise ValueError("Q8_0 needs whole 32-element blocks")
        self._ptr = check_ptr(lib().llamd_hip_upload_q8_0(_ptr(w), rows, k), "upload_q8_0")
        self.rows, self.k = rows, k

    def matvec(self, x) -> np.ndarray:
        x = _f32(x)
        if x.size != self.k:
            raise ValueError(f"expected {self.k} activations, got {x.size}")
        out = np.empty(self.rows, np.float32)
        check(lib().llamd_hip_matvec_q8_0(self._ptr, _ptr(x), _ptr(out), self.rows, self.k),
              "matvec_q8_0")
        return out

    def dequantize(self) -> np.ndarray:
        out = np.empty((self.rows, self.k), np.float32)
        check(lib().llamd_hip_dequant_q8_0(self._ptr, self.rows, self.k, _ptr(out)), "dequant_q8_0")
        return out

    def close(self):
        if self._ptr:
            lib().llamd_rocm_release(self._ptr)
            self._ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def matvec_q6k(w, act: BlockQ8K, rows: int) -> np.ndarray:
    """Upload, multiply, release (crates/llamd-rocm/src/lib.rs:914-)."""
    blocks = act.nblocks
    dw = DeviceWeights.upload(w, rows, blocks)
    try:
        return dw.matvec(act)
    finally:
        dw.close()


@dataclass
class Routing:
    experts: np.ndarray   # int32 [n_used], best first
    weights: np.ndarray   # f32 [n_used], renormalised


def route(logits, n_used: int) -> Routing:
    """crates/llamd-models/src/moe.rs:73-113 on the device."""
    lg = _f32(logits)
    if n_used == 0 or n_used > lg.size:
        raise ValueError(f"{n_used} experts requested of {lg.size}")
    ids = np.empty(n_used, np.int32)
    w = np.empty(n_used, np.float32)
    check(lib().llamd_hip_route(_ptr(lg), lg.size, n_used, _ptr(ids), _ptr(w)), "route")
    return Routing(ids, w)


SAMPLING = np.dtype([("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32)])


def sampling_rules(n_seq: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> np.ndarray:
    """llamd_hip_sampling [n_seq] from numbers or arrays of one per sequence."""
    r = np.zeros(n_seq, SAMPLING)
    for name, x in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if np.ndim(x) > 1 or (np.ndim(x) == 1 and len(x) != n_seq):
            raise ValueError(f"{name}: one number, or one per sequence")
        if name == "top_k":
            k = np.asarray(x, np.float64)
            if not ((k == np.rint(k)) & (np.abs(k + 0.5) < 2.0 ** 31)).all():
                raise ValueError("top_k: whole numbers of 32 bits")
        r[name] = x
    return r


def _sample_device(logits_ptr, ld: int, n: int, rules: np.ndarray, u) -> tuple[np.ndarray, np.ndarray]:
    """(ids, probabilities) of rows of device logits."""
    n_seq = len(rules)
    u = np.ascontiguousarray(np.broadcast_to(np.asarray(u, np.float64), (n_seq,)))
    ids, prob = np.empty(n_seq, np.int32), np.empty(n_seq, np.float32)
    if not n_seq:
        return ids, prob
    how, du = DeviceBuffer.from_array(rules), DeviceBuffer.from_array(u)
    di, dp = DeviceBuffer(ids.nbytes), DeviceBuffer(prob.nbytes)
    check(lib().llamd_hip_sample(logits_ptr, ld, n, n_seq, how.ptr, du.ptr, di.ptr, dp.ptr), "sample")
    return di.download(ids), dp.download(prob)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> tuple[np.ndarray, np.ndarray]:
    """A token per row of logits [n_seq, n] and the probability that it was drawn with (llamd_hip_sample): u uniform
    numbers in [0, 1), one per row; the rule's numbers for all rows or one per row."""
    x = np.atleast_2d(_f32(logits))
    if x.ndim > 2:
        raise ValueError("logits must be [n_seq, n]")
    if np.shape(u) not in ((), (len(x),)):
        raise ValueError("u: one number per row")
    rules = sampling_rules(len(x), temperature, top_k, top_p, min_p)
    if not x.size:
        raise ValueError("no logits")
    dx = DeviceBuffer.from_array(x)  # (held until the results are back)
    return _sample_device(dx.ptr, x.shape[1], x.shape[1], rules, u)


def argmax(x) -> np.ndarray:
    """Row-wise argmax, lowest index on ties."""
    x = np.atleast_2d(_f32(x))
    ids = np.empty(x.shape[0], np.int32)
    check(lib().llamd_hip_argmax(_ptr(x), x.shape[1], x.shape[0], _ptr(ids)), "argmax")
    return ids


class MoeLayer:
    """One MoE FFN (router -> route -> experts -> combine) resident on the device.

    router: f32 [n_expert, n_embd]; gate/up: ggml Q6_K bytes of
    [n_expert][n_ff][n_embd]; down: [n_expert][n_embd][n_ff]."""

    EXACT = 1

    def __init__(self, router, gate, up, down, n_embd: int, n_ff: int, n_expert: int, n_used: int):
        router = _f32(router)
        gate, up, down = (np.ascontiguousarray(a, dtype=np.uint8) for a in (gate, up, down))
        if router.size != n_expert * n_embd:
            raise ValueError("router must be [n_expert, n_embd]")
        per = n_ff * n_embd // QK_K * Q6K_BLOCK_BYTES
        if gate.size < n_expert * per or up.size < n_expert * per or down.size < n_expert * per:
            raise ValueError("expert tensors are short")
        self.n_embd, self.n_ff, self.n_expert, self.n_used = n_embd, n_ff, n_expert, n_used
        self._h = check_ptr(lib().llamd_hip_moe_create(_ptr(router), _ptr(gate), _ptr(up), _ptr(down),
                                                       n_embd, n_ff, n_expert, n_used), "moe_create")

    @classmethod
    def from_handle(cls, h, n_embd: int, n_ff: int, n_expert: int, n_used: int) -> "MoeLayer":
        """Wrap a layer the library built elsewhere (e.g. llamd_gguf_moe_create)."""
        m = cls.__new__(cls)
        m.n_embd, m.n_ff, m.n_expert, m.n_used = n_embd, n_ff, n_expert, n_used
        m._h = check_ptr(h, "moe layer")
        return m

    @property
    def handle(self):
        return self._h

    def forward(self, x, res=None, exact: bool = True):
        """Returns (out, Routing, logits). out = res + moe_ffn(x) (res optional).
        Every call is bit-exact; `exact` is accepted for older callers."""
        x = _f32(x)
        if x.size != self.n_embd:
            raise ValueError("x must be [n_embd]")
        r = None if res is None else _f32(res)
        out = np.empty(self.n_embd, np.float32)
        ids = np.empty(self.n_used, np.int32)
        w = np.empty(self.n_used, np.float32)
        lg = np.empty(self.n_expert, np.float32)
        check(lib().llamd_hip_moe_forward_host(self._h, _ptr(x), _ptr(r), _ptr(out), _ptr(ids),
                                               _ptr(w), _ptr(lg), self.EXACT if exact else 0),
              "moe_forward")
        return out, Routing(ids, w), lg

    def forward_batch(self, x, res=None):
        """nseq sequences at once, each routed by its own logits; returns
        (out [nseq, n_embd], ids [nseq, n_used], weights [nseq, n_used],
        logits [nseq, n_expert]). Bit-identical to forward() per row."""
        x = _f32(x).reshape(-1, self.n_embd)
        nseq = x.shape[0]
        r = None if res is None else _f32(res).reshape(nseq, self.n_embd)
        out = np.empty((nseq, self.n_embd), np.float32)
        ids = np.empty((nseq, self.n_used), np.int32)
        w = np.empty((nseq, self.n_used), np.float32)
        lg = np.empty((nseq, self.n_expert), np.float32)
        check(lib().llamd_hip_moe_forward_batch_host(self._h, _ptr(x), _ptr(r), _ptr(out), _ptr(ids),
                                                     _ptr(w), _ptr(lg), nseq), "moe_forward_batch")
        return out, ids, w, lg

    def prefill(self, x, ids, weights, reduction: bool = False) -> np.ndarray:
        """moe_ffn for n_tok tokens with the given routing [n_tok, n_used].
        reduction=True: the REDUCTION-tolerance GEMMs (LLAMD_HIP_REDUCTION);
        otherwise bit-identical to the CPU path."""
        x = _f32(x).reshape(-1, self.n_embd)
        n_tok = x.shape[0]
        ids = np.ascontiguousarray(ids, dtype=np.int32).reshape(n_tok, self.n_used)
        w = _f32(weights).reshape(n_tok, self.n_used)
        out = np.empty((n_tok, self.n_embd), np.float32)
        check(lib().llamd_hip_moe_prefill_host_ex(self._h, _ptr(x), _ptr(ids), _ptr(w), _ptr(out), n_tok,
                                                  1 if reduction else 0), "moe_prefill")
        return out

    def stats(self) -> tuple[int, int]:
        a, b = C.c_int(), C.c_int()
        check(lib().llamd_hip_moe_stats(self._h, C.byref(a), C.byref(b)), "moe_stats")
        return a.value, b.value

    def counters(self) -> tuple[np.ndarray, np.ndarray]:
        """([calls, exact calls, certified calls, wait timed out], the last
        call's logit estimates T [n_expert] and bounds E [n_expert])."""
        c = np.zeros(4, np.int32)
        est = np.zeros(2 * self.n_expert, np.float64)
        check(lib().llamd_hip_moe_counters(self._h, c.ctypes.data_as(C.POINTER(C.c_int)), _ptr(est)),
              "moe_counters")
        return c, est.reshape(2, self.n_expert)

    def close(self):
        if self._h:
            lib().llamd_hip_moe_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DeviceBuffer:
    """Raw device memory on the library's allocator (for device-pointer calls)."""

    def __init__(self, nbytes: int):
        self.nbytes = nbytes
        self.ptr = check_ptr(lib().llamd_fwd_alloc(nbytes), "alloc")

    @classmethod
    def from_array(cls, a: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(a)
        b = cls(a.nbytes)
        b.upload(a)
        return b

    def upload(self, a: np.ndarray):
        a = np.ascontiguousarray(a)
        if a.nbytes > self.nbytes:
            raise ValueError("array larger than buffer")
        check(lib().llamd_fwd_upload(self.ptr, _ptr(a), a.nbytes), "upload")

    def download(self, a: np.ndarray) -> np.ndarray:
        if a.nbytes > self.nbytes:
            raise ValueError("array larger than buffer")
        check(lib().llamd_fwd_download(_ptr(a), self.ptr, a.nbytes), "download")
        return a

    def close(self):
        if self.ptr:
            lib().llamd_fwd_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class LmHead:
    """Q6_K output projection + argmax over the vocabulary."""

    def __init__(self, weights: DeviceWeights, max_seq: int = 16):
        self.w = weights
        self.rows, self.blocks, self.max_seq = weights.rows(), weights.blocks(), max_seq
        self._h = check_ptr(lib().llamd_hip_lmhead_create(weights.ptr, self.rows, self.blocks, max_seq),
                            "lmhead_create")
        self._x = DeviceBuffer(max_seq * self.blocks * QK_K * 4)
        self._logits = DeviceBuffer(max_seq * self.rows * 4)
        self._ids = DeviceBuffer(max_seq * 4)

    @property
    def handle(self):
        return self._h

    def forward(self, x, reduction: bool = False) -> tuple[np.ndarray, np.ndarray]:
        """logits [nseq, rows] and arg-max ids [nseq]. reduction=True
        (LLAMD_HIP_REDUCTION, nseq > 1): logits within REDUCTION, ids still
        the exact logits' arg-max."""
        x = np.atleast_2d(_f32(x))
        nseq = x.shape[0]
        if x.shape[1] != self.blocks * QK_K or nseq > self.max_seq:
            raise ValueError("x must be [nseq <= max_seq, k]")
        self._x.upload(x)
        check(lib().llamd_hip_lmhead_forward_ex(self._h, self._x.ptr, nseq, self._logits.ptr, self._ids.ptr,
                                                1 if reduction else 0), "lmhead_forward")
        logits = self._logits.download(np.empty((nseq, self.rows), np.float32))
        ids = self._ids.download(np.empty(nseq, np.int32))
        return logits, ids

    def sample(self, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> tuple[np.ndarray, np.ndarray]:
        """A drawn token per sequence and its probability (sample), from logits that stay on the device."""
        x = np.atleast_2d(_f32(x))
        nseq = x.shape[0]
        if x.ndim > 2 or x.shape[1] != self.blocks * QK_K or not 0 < nseq <= self.max_seq:
            raise ValueError("x must be [1 <= nseq <= max_seq, k]")
        if np.shape(u) not in ((), (nseq,)):
            raise ValueError("u: one number per sequence")
        rules = sampling_rules(nseq, temperature, top_k, top_p, min_p)
        self._x.upload(x)
        check(lib().llamd_hip_lmhead_forward(self._h, self._x.ptr, nseq, self._logits.ptr, self._ids.ptr), "lmhead_forward")
        return _sample_device(self._logits.ptr, self.rows, self.rows, rules, u)

    def close(self):
        if self._h:
            lib().llamd_hip_lmhead_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Pages(C.Structure):
    """llamd_hip_pages: a paged cache's memory. k [n_page][n_head_kv][page][hd],
    v [n_page][n_head_kv][hd][page]; type is ggml's number (PAGE_TYPES)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("type", C.c_int), ("n_page", C.c_int),
                ("page", C.c_int), ("n_head_kv", C.c_int), ("hd", C.c_int)]


class Pages8(C.Structure):
    """llamd_hip_pages8: an 8-bit paged cache's memory. k and v as in Pages, bytes; a
    scale byte for each 16 positions of a page and kv head."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("n_page", C.c_int),
                ("page", C.c_int), ("n_head_kv", C.c_int), ("hd", C.c_int)]


class Batch(C.Structure):
    """llamd_hip_batch: the packed tokens of a call (device pointers)."""
    _fields_ = [("start", C.c_void_p), ("len", C.c_void_p), ("table", C.c_void_p),
                ("n_seq", C.c_int), ("n_tok", C.c_int), ("max_page", C.c_int)]


PAGE_TYPES = {"f32": 0, "f16": 1, "bf16": 30}


def to_bf16(x) -> np.ndarray:
    """f32 -> bf16 bits (uint16), rounded to nearest even."""
    u = _f32(x).view(np.uint32)
    nan = np.isnan(_f32(x))
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), r)


def from_bf16(b) -> np.ndarray:
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _e4m3_values() -> np.ndarray:
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    x = np.where(e, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    x[127] = x[255] = np.nan
    return np.where(b < 128, x, -x).astype(np.float32)


_E4M3 = _e4m3_values()


def from_e4m3(b) -> np.ndarray:
    return _E4M3[np.asarray(b, np.uint8)]


def to_e4m3(x) -> np.ndarray:
    """Values of up to 448 -> e4m3 bytes, rounded to nearest even; NaN for what is larger or not finite."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, np.inf))
    step = 2.0 ** (np.clip(np.frexp(np.where(np.isinf(a), 0, a))[1] - 1, -6, 8) - 3)
    a = np.rint(np.minimum(a, 1e9) / step) * step
    code = np.searchsorted(_E4M3[:127], a.astype(np.float32)).clip(0, 126)
    return (np.where(a > 448, 127, code) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_byte(top) -> np.ndarray:
    """The scale byte of 16 positions whose largest magnitude is `top`: the least E, 1 to 254, with top <= 448 * 2^(E - 127)."""
    m, e = np.frexp(_f32(top))  # top = m 2^e, m in [1/2, 1)
    return np.where(_f32(top) > 0, np.clip(127 + e - 9 + (m > 0.875), 1, 254), 1).astype(np.uint8)


def rope_freqs(n_rot: int, base: float, factor: float = 1.0, orig_ctx: int = 0, beta_fast: float = 32.0,
               beta_slow: float = 1.0) -> tuple[np.ndarray, float]:
    """(radians per position [n_rot / 2] f64, magnitude): llamd_hip_rope_freqs."""
    f = np.empty(max(n_rot, 2) // 2, np.float64)
    m = C.c_float()
    check(lib().llamd_hip_rope_freqs(n_rot, base, factor, orig_ctx, beta_fast, beta_slow, _ptr(f), C.byref(m)),
          "rope_freqs")
    return f, m.value


class PagedCache:
    """One layer's paged KV cache (llamd_hip_paged_*) with host arrays in and
    out. A batch is (table [n_seq, max_page], length [n_seq], start [n_seq + 1]
    or None for one token each); q and results cross as f32. A program that
    keeps its data on the device fills Pages and Batch and calls the C ABI."""

    calls = "llamd_hip_paged"

    def __init__(self, type: str, n_page: int, page: int, n_head: int, n_head_kv: int, hd: int):
        if type not in PAGE_TYPES:
            raise ValueError(f"type {type!r}: f32, f16 or bf16")
        if min(n_page, page, n_head_kv, hd) <= 0:
            raise ValueError("n_page, page, n_head_kv and hd must be positive")
        self.type, self.n_head = type, n_head
        self.dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[type]
        self.shape_k, self.shape_v = (n_page, n_head_kv, page, hd), (n_page, n_head_kv, hd, page)
        zero = np.zeros(self.shape_k, self.dtype)
        self._k, self._v = DeviceBuffer.from_array(zero), DeviceBuffer.from_array(zero)
        self.pages = Pages(self._k.ptr, self._v.ptr, PAGE_TYPES[type], n_page, page, n_head_kv, hd)

    def encode(self, x) -> np.ndarray:
        return to_bf16(x) if self.type == "bf16" else _f32(x).astype(self.dtype)

    def decode_values(self, x) -> np.ndarray:
        return from_bf16(x) if self.type == "bf16" else x.astype(np.float32)

    def read(self) -> tuple[np.ndarray, np.ndarray]:
        """(K, V) pages as f32."""
        k = self._k.download(np.empty(self.shape_k, self.dtype))
        v = self._v.download(np.empty(self.shape_v, self.dtype))
        return self.decode_values(k), self.decode_values(v)

    def write(self, k, v):
        k, v = self.encode(k), self.encode(v)
        if k.shape != self.shape_k or v.shape != self.shape_v:
            raise ValueError(f"pages are {self.shape_k} and {self.shape_v}")
        self._k.upload(k)
        self._v.upload(v)

    def _batch(self, table, length, start, n_tok):
        table = np.ascontiguousarray(np.atleast_2d(table), np.int32)
        length = np.ascontiguousarray(length, np.int32)
        if table.shape[0] != length.size or (start is not None and len(start) != length.size + 1):
            raise ValueError("one table row, length and start per sequence")
        keep = [DeviceBuffer.from_array(length), DeviceBuffer.from_array(table)]
        if start is not None:
            keep.append(DeviceBuffer.from_array(np.ascontiguousarray(start, np.int32)))
        b = Batch(keep[2].ptr if start is not None else None, keep[0].ptr, keep[1].ptr, length.size, n_tok,
                  table.shape[1])
        return b, keep

    def store(self, q, k, v, table, length, start=None, q_norm=None, k_norm=None, eps: float = 1e-6, freqs=None,
              interleaved: bool = False, mscale: float = 1.0) -> np.ndarray:
        """q [n_tok, n_head * hd], k, v [n_tok, n_head_kv * hd]; the rotated q
        (f32 values of the cache's type), k and v in the pages."""
        _, kvh, _, hd = self.shape_k
        q, k, v = _f32(q), _f32(k), _f32(v)
        if q.shape[1:] != (self.n_head * hd,) or k.shape != (q.shape[0], kvh * hd) or v.shape != k.shape:
            raise ValueError("q must be [n_tok, n_head * hd], k and v [n_tok, n_head_kv * hd]")
        for w in (q_norm, k_norm):
            if w is not None and np.size(w) != hd:
                raise ValueError("norm weights must be [hd]")
        b, keep = self._batch(table, length, start, q.shape[0])
        dev = [DeviceBuffer.from_array(x) for x in (q, k, v)]
        norms = [None if w is None else DeviceBuffer.from_array(_f32(w)) for w in (q_norm, k_norm)]
        fr = None if freqs is None else DeviceBuffer.from_array(np.ascontiguousarray(freqs, np.float64))
        out = DeviceBuffer.from_array(np.zeros(q.shape, self.dtype))
        check(getattr(lib(), self.calls + "_store")(
            C.byref(self.pages), C.byref(b), dev[0].ptr, self.n_head * hd, dev[1].ptr, kvh * hd, dev[2].ptr, kvh * hd,
            *(None if w is None else w.ptr for w in norms), eps, fr and fr.ptr,
            0 if freqs is None else 2 * len(freqs), int(interleaved), mscale, self.n_head, out.ptr), "paged_store")
        return self.decode_values(out.download(np.empty(q.shape, self.dtype)))

    def _attend(self, call, q, table, length, start, scale, f32_out):
        hd = self.shape_k[3]
        q = self.encode(q)
        if q.ndim != 2 or q.shape[1] != self.n_head * hd:
            raise ValueError("q must be [n_tok, n_head * hd]")
        b, keep = self._batch(table, length, start, q.shape[0])
        dq = DeviceBuffer.from_array(q)
        dtype = np.float32 if f32_out else self.dtype
        out = DeviceBuffer.from_array(np.zeros(q.shape, dtype))
        call(b, dq, hd ** -0.5 if scale is None else scale, 0 if f32_out else PAGE_TYPES[self.type], out)
        got = out.download(np.empty(q.shape, dtype))
        return got if f32_out else self.decode_values(got)

    def prompt(self, q, table, length, start, scale: float | None = None, f32_out: bool = False) -> np.ndarray:
        """Causal attention of the packed tokens q [n_tok, n_head * hd]."""
        def call(b, dq, scale, number, out):
            check(getattr(lib(), self.calls + "_prompt")(C.byref(self.pages), C.byref(b), dq.ptr, self.n_head, scale, number,
                                                         out.ptr), "paged_prompt")
        return self._attend(call, q, table, length, start, scale, f32_out)

    def decode(self, q, table, length, group=None, shared=None, scale: float | None = None,
               f32_out: bool = False) -> np.ndarray:
        """One token per sequence; group [n_group + 1] first sequences and
        shared [n_group] positions where sequences share a prefix."""
        if (group is None) != (shared is None) or (group is not None and len(group) != len(shared) + 1):
            raise ValueError("group and shared go together, one more first sequence than groups")
        g = None if group is None else [DeviceBuffer.from_array(np.ascontiguousarray(x, np.int32))
                                        for x in (group, shared)]

        def call(b, dq, scale, number, out):
            check(getattr(lib(), self.calls + "_decode")(C.byref(self.pages), C.byref(b), g and g[0].ptr, g and g[1].ptr,
                                                         0 if g is None else len(shared), dq.ptr, self.n_head, scale, number,
                                                         out.ptr), "paged_decode")
        return self._attend(call, q, table, length, None, scale, f32_out)

    def close(self):
        self._k.close()
        self._v.close()


class PagedCache8(PagedCache):
    """One layer's 8-bit paged KV cache (llamd_hip_paged8_*): e4m3 numbers with a power of two for each 16 positions
    of a page and kv head. q and results are bf16 values."""

    calls = "llamd_hip_paged8"

    def __init__(self, n_page: int, page: int, n_head: int, n_head_kv: int, hd: int):
        if min(n_page, page, n_head_kv, hd) <= 0 or page % 16:
            raise ValueError("n_page, page, n_head_kv and hd must be positive, page a multiple of 16")
        self.type, self.n_head, self.dtype = "bf16", n_head, np.uint16
        self.shape_k, self.shape_v = (n_page, n_head_kv, page, hd), (n_page, n_head_kv, hd, page)
        self.shape_scale = (n_page, n_head_kv, page // 16)
        self._k, self._v = (DeviceBuffer.from_array(np.zeros(self.shape_k, np.uint8)) for _ in range(2))
        self._ks, self._vs = (DeviceBuffer.from_array(np.ones(self.shape_scale, np.uint8)) for _ in range(2))
        self.pages = Pages8(self._k.ptr, self._v.ptr, self._ks.ptr, self._vs.ptr, n_page, page, n_head_kv, hd)

    def read_bytes(self) -> tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
        """(K, V, K's scales, V's scales) as they lie in memory."""
        return tuple(b.download(np.empty(shape, np.uint8)) for b, shape in (
            (self._k, self.shape_k), (self._v, self.shape_v), (self._ks, self.shape_scale), (self._vs, self.shape_scale)))

    def write_bytes(self, k, v, k_scale, v_scale):
        for b, x, shape in ((self._k, k, self.shape_k), (self._v, v, self.shape_v), (self._ks, k_scale, self.shape_scale),
                            (self._vs, v_scale, self.shape_scale)):
            if np.shape(x) != shape:
                raise ValueError(f"pages are {self.shape_k} and {self.shape_v}, scales {self.shape_scale}")
            b.upload(np.ascontiguousarray(x, np.uint8))

    def read(self) -> tuple[np.ndarray, np.ndarray]:
        """(K, V) pages as f32."""
        k, v, ks, vs = self.read_bytes()
        unit = [np.exp2(np.repeat(np.maximum(s, 1).astype(np.float32), 16, 2) - 127) for s in (ks, vs)]
        return from_e4m3(k) * unit[0][..., None], from_e4m3(v) * unit[1][:, :, None, :]

    def write(self, k, v):
        """f32 pages; each 16 positions get the scale that their largest finite value needs."""
        if np.shape(k) != self.shape_k or np.shape(v) != self.shape_v:
            raise ValueError(f"pages are {self.shape_k} and {self.shape_v}")
        n_page, kvh, page, hd = self.shape_k
        k = _f32(k).reshape(n_page, kvh, page // 16, 16 * hd)
        v = _f32(v).reshape(n_page, kvh, hd, page // 16, 16)
        top = [np.where(np.isfinite(x), np.abs(x), 0).max(axis) for x, axis in ((k, 3), (v, (2, 4)))]
        ks, vs = (scale_byte(t) for t in top)
        unit = [np.exp2(127 - s.astype(np.float64)) for s in (ks, vs)]
        self.write_bytes(to_e4m3(k * unit[0][..., None]).reshape(self.shape_k),
                         to_e4m3(v * unit[1][:, :, None, :, None]).reshape(self.shape_v), ks, vs)

    def close(self):
        super().close()
        self._ks.close()
        self._vs.close()


__all__ = [
    "Pages", "Pages8", "Batch", "PagedCache", "PagedCache8", "PAGE_TYPES", "rope_freqs", "to_bf16", "from_bf16", "to_e4m3",
    "from_e4m3", "scale_byte", "SAMPLING", "sampling_rules", "sample",
    "BlockQ8K", "DeviceInfo", "DeviceWeights", "Q8_0Weights", "MoeLayer", "LmHead", "Routing",
    "DeviceBuffer", "available", "device_count", "device_info", "quantize_q8k_on_device",
    "swiglu_q8k_on_device", "matvec_q6k", "route", "argmax", "HipError", "HipUnavailable",
]


class _PinnedPool:
    """Page-locked host buffers of one size (hipHostMalloc), handed out as
    numpy arrays and taken back when an array is collected. A device-to-host
    copy into page-locked memory is one DMA, without the bounce buffer a
    pageable destination goes through (608 KB of logits: ~48 us -> ~12 us)."""

    def __init__(self, nbytes: int):
        self.nbytes = nbytes
        self._free = []
        self._closed = False
        hip = C.CDLL("libamdhip64.so.7")   # already loaded by the library
        self._malloc = hip.hipHostMalloc
        self._malloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t, C.c_uint]
        self._malloc.restype = C.c_int
        self._hfree = hip.hipHostFree
        self._hfree.argtypes = [C.c_void_p]
        self._hfree.restype = C.c_int

    def _put(self, ptr):
        if self._closed:
            self._hfree(ptr)
        else:
            self._free.append(ptr)

    def array(self, n: int, dtype) -> np.ndarray:
        if self._free:
            ptr = self._free.pop()
        else:
            p = C.c_void_p()
            if self._malloc(C.byref(p), self.nbytes, 0) != 0 or not p.value:
                raise HipError("hipHostMalloc failed")
            ptr = p.value
        arr = np.frombuffer((C.c_char * self.nbytes).from_address(ptr), dtype=dtype, count=n)
        fin = weakref.finalize(arr, self._put, ptr)
        fin.atexit = False  # at interpreter exit the process's pages go with it
        return arr

    def close(self):
        self._closed = True
        while self._free:
            self._hfree(self._free.pop())


class DeviceModel:
    """A resident Qwen3-MoE decode loop from a GGUF (DeviceModel::load /
    forward, crates/llamd-runtime/src/device.rs:262-722): weights uploaded
    once, KV cache for max_kv positions, one synchronisation per token."""

    def __init__(self, gguf, max_kv: int):
        self._h = check_ptr(lib().llamd_hip_model_create(gguf._h, max_kv), "model_create")
        a, b, c, d = C.c_int(), C.c_int(), C.c_int(), C.c_int()
        check(lib().llamd_hip_model_info(self._h, C.byref(a), C.byref(b), C.byref(c), C.byref(d)),
              "model_info")
        self.n_layer, self.n_embd, self.n_vocab, self.max_kv = a.value, b.value, c.value, d.value
        self._pinned = _PinnedPool(self.n_vocab * 4)

    def forward(self, token: int, pos: int):
        """(logits [n_vocab], next token = argmax) for `token` at `pos`. The
        logits live in page-locked host memory (returned to a pool when the
        array is collected)."""
        logits = self._pinned.array(self.n_vocab, np.float32)
        nxt = np.zeros(1, np.int32)
        check(lib().llamd_hip_model_forward(self._h, int(token), int(pos), _ptr(logits), _ptr(nxt)),
              "model_forward")
        return logits, int(nxt[0])

    def close(self):
        if self._h:
            lib().llamd_hip_model_destroy(self._h)
            self._h = None
        if getattr(self, "_pinned", None) is not None:
            self._pinned.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
