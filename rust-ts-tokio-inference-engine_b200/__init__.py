"""Host-side binding of the B200 ragged hybrid-Qwen decode step.

The product is the C-ABI library ``_lib/libqwen_b200.so`` (CUDA, sm_100a). This
module binds it with ctypes the same way the reference's Rust executor binds
its native bridge (src/serving/native_device.rs:1087-1207): same symbols, same
argument meaning, and the same error convention (0 = ok, -1 = error with a
message, surfaced here as ``NativeError``). There is no CPU path: loading
fails loudly when the library is missing, and creating a session fails on a
machine without a B200.
"""
from __future__ import annotations

import ctypes as C
import struct
from pathlib import Path

import numpy as np

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "_lib" / "libqwen_b200.so"

RAGGED_SAMPLED = 1
RAGGED_LOGITS = 2
RAGGED_ALL_ROWS = 4
RAGGED_HIDDEN = 8
RAGGED_CONSUME = 16
STATS_COUNT = 17 + 19 * 3


class NativeError(RuntimeError):
    """A native call returned -1 (native/mlx_bridge.cpp:19-31 convention)."""


class RsQwenConfig(C.Structure):
    """rs_qwen_config (native/mlx_bridge.h:50-53)."""

    _fields_ = [(n, C.c_int32) for n in (
        "hidden layers vocab q_heads kv_heads head_dim key_heads value_heads key_dim "
        "value_dim conv interval experts top intermediate shared group bits context chunk "
        "rope_dims activation_precision layer_group fused_recurrent execution_timing "
        "compiled_decode operator_profile fused_attention validation_mode "
        "validation_interval expert_kernel").split()] + [("epsilon", C.c_float), ("theta", C.c_float)]


class RsQwenLayer(C.Structure):
    _fields_ = [("index", C.c_uint32), ("mixer", C.c_uint32)]


class StateId(C.Structure):
    """StateId {owner, slot, generation, position, bytes} (native/state_table.h:11-13)."""

    _fields_ = [(n, C.c_uint64) for n in ("owner", "slot", "generation", "position", "bytes")]

    def astuple(self):
        return (self.owner, self.slot, self.generation, self.position, self.bytes)


class Kv4CacheDesc(C.Structure):
    """rs_qwen_kv4_cache."""

    _fields_ = [(n, C.c_int32) for n in ("device", "q_heads", "kv_heads", "head_dim")] + [
        ("pages", C.c_uint64), ("pool", C.c_void_p), ("status", C.c_void_p)]


class Kv4Rows(C.Structure):
    """rs_qwen_kv4_rows."""

    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class Kv4AppendArgs(C.Structure):
    """rs_qwen_kv4_append_args."""

    _fields_ = [("q", Kv4Rows), ("k", Kv4Rows), ("v", Kv4Rows), ("dtype", C.c_uint32), ("q_out_dtype", C.c_uint32),
                ("tokens", C.c_size_t), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("positions", C.c_void_p),
                ("slots", C.c_void_p), ("q_out", C.c_void_p), ("epsilon", C.c_float), ("theta", C.c_float),
                ("rope_dims", C.c_int32), ("reserved", C.c_int32)]


class Kv4AttentionArgs(C.Structure):
    """rs_qwen_kv4_attention_args."""

    _fields_ = [("q", Kv4Rows), ("gate", Kv4Rows), ("out", Kv4Rows), ("dtype", C.c_uint32), ("reserved", C.c_uint32),
                ("n_seq", C.c_size_t), ("tokens", C.c_size_t), ("max_count", C.c_size_t), ("cu_seqlens", C.c_void_p),
                ("kv_lens", C.c_void_p), ("block_table", C.c_void_p), ("table_stride", C.c_int64), ("scale", C.c_float),
                ("lse", C.c_void_p), ("weights_in", C.c_void_p), ("weights_out", C.c_void_p),
                ("weights_stride", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class Kv4EvictArgs(C.Structure):
    """rs_qwen_kv4_evict_args."""

    _fields_ = [("n_seq", C.c_size_t), ("kv_lens", C.c_void_p), ("src_table", C.c_void_p), ("src_stride", C.c_int64),
                ("dst_table", C.c_void_p), ("dst_stride", C.c_int64), ("weights", C.c_void_p),
                ("weights_stride", C.c_int64), ("keep", C.c_int32), ("recent", C.c_int32), ("kept", C.c_void_p),
                ("new_lens", C.c_void_p), ("weights_out", C.c_void_p), ("weights_out_stride", C.c_int64)]


assert C.sizeof(RsQwenConfig) == 132 and C.sizeof(StateId) == 40

_P, _SZ, _U32P, _F32P, _I32P = C.c_void_p, C.c_size_t, C.POINTER(C.c_uint32), C.POINTER(C.c_float), C.POINTER(C.c_int32)
_SIDP, _ERR = C.POINTER(StateId), C.c_char_p

# symbol -> (restype, argtypes); the declarations of include/qwen_b200.h
SIGNATURES = {
    "rs_mlx_version": (C.c_char_p, []),
    "rs_qwen_state_count": (_SZ, [C.POINTER(RsQwenConfig)]),
    "rs_mlx_weights_create": (_P, [_ERR, _SZ]),
    "rs_mlx_weights_destroy": (None, [_P]),
    "rs_mlx_weights_load": (C.c_int, [_P, C.c_char_p, _ERR, _SZ]),
    "rs_qwen_quant": (C.c_int, [_P, C.c_char_p, C.c_int, C.c_int, _ERR, _SZ]),
    "rs_mlx_weight_bytes": (C.c_int, [_P, C.c_char_p, _I32P, _SZ, C.c_int, _SZ, C.POINTER(C.c_uint8), _SZ, _ERR, _SZ]),
    "rs_qwen_weights_synthetic": (C.c_int, [_P, C.POINTER(RsQwenConfig), C.c_uint64, C.c_int, _ERR, _SZ]),
    "rs_qwen_forward": (C.c_int, [_P, C.c_int, C.POINTER(RsQwenConfig), C.POINTER(RsQwenLayer), _SZ, _U32P, _SZ, _SZ,
                                  _F32P, _SZ, _F32P, _SZ, _F32P, _SZ, C.c_int, _U32P, _SZ, _F32P, _SZ, _ERR, _SZ]),
    "rs_mlx_create": (_P, [C.c_int, _ERR, _SZ]),
    "rs_mlx_destroy": (None, [_P]),
    "rs_mlx_input": (C.c_int, [_P, C.c_int, C.c_void_p, _I32P, _SZ, _ERR, _SZ]),
    "rs_mlx_op": (C.c_int, [_P, C.c_int, _U32P, _SZ, C.c_int, C.c_float, _ERR, _SZ]),
    "rs_mlx_finish": (C.c_int, [_P, C.c_uint32, C.c_void_p, _SZ, _ERR, _SZ]),
    "rs_mlx_kernel": (C.c_int, [_P, C.c_int, _U32P, _SZ, _I32P, _SZ, _F32P, _SZ, _ERR, _SZ]),
    "rs_mlx_parameter": (C.c_int, [_P, _P, C.c_char_p, _I32P, _SZ, C.c_int, _ERR, _SZ]),
    "rs_mlx_cleanup": (None, []),
    "rs_qwen_device_create": (_P, [_P, C.c_int, C.POINTER(RsQwenConfig), C.POINTER(RsQwenLayer), _SZ, _SZ,
                                   C.c_uint64, _ERR, _SZ]),
    "rs_qwen_device_destroy": (None, [_P]),
    "rs_qwen_device_decode_batch": (C.c_int, [_P, _SIDP, _U32P, _SZ, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_step": (C.c_int, [_P, _SIDP, _SZ, _U32P, _SZ, _SIDP, _F32P, _SZ, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_step_sampled": (C.c_int, [_P, _SIDP, _SZ, _U32P, _SZ, _SIDP, _U32P, _ERR, _SZ]),
    "rs_qwen_device_block": (C.c_int, [_P, _SIDP, _SZ, _U32P, _SZ, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_hidden_step": (C.c_int, [_P, _SIDP, _SZ, _U32P, _SZ, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_hidden_block": (C.c_int, [_P, _SIDP, _SZ, _U32P, _SZ, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_hidden_snapshot": (C.c_int, [_P, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_release": (C.c_int, [_P, _SIDP, _ERR, _SZ]),
    "rs_qwen_device_snapshot": (C.c_int, [_P, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_stats": (C.c_int, [_P, C.POINTER(C.c_uint64), _SZ, _ERR, _SZ]),
    "rs_qwen_device_drain": (C.c_int, [_P, C.POINTER(C.c_uint64), _ERR, _SZ]),
    "rs_qwen_device_mtp_attach": (C.c_int, [_P, _P, _ERR, _SZ]),
    "rs_qwen_device_mtp_step": (C.c_int, [_P, _SIDP, _SIDP, C.c_int, _SZ, _U32P, _SZ, _SIDP, _F32P, _SZ,
                                          C.c_int, _ERR, _SZ]),
    "rs_qwen_device_mtp_release": (C.c_int, [_P, _SIDP, _ERR, _SZ]),
    "rs_qwen_device_mtp_snapshot": (C.c_int, [_P, _SIDP, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_step_ragged": (C.c_int, [_P, _SZ, _SIDP, _U32P, _U32P, _U32P, C.c_uint32, _SIDP, _U32P, _SZ,
                                             _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_step_ragged_choices": (C.c_int, [_P, _SZ, _SIDP, _U32P, _U32P, _U32P, C.c_uint32, _U32P, _U32P,
                                                     _SZ, _SIDP, _U32P, _SZ, _F32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_mtp_verify_accept": (C.c_int, [_P, _SZ, _SIDP, _U32P, _U32P, _U32P, _SZ, _U32P, _SZ,
                                                   C.c_uint32, _SIDP, _U32P, _U32P, _U32P, _ERR, _SZ]),
    "rs_qwen_device_synthetic_state": (C.c_int, [_P, _SZ, C.c_uint64, _SIDP, _ERR, _SZ]),
    "rs_qwen_device_kv4": (C.c_int, [_P, C.c_int, _ERR, _SZ]),
    "rs_qwen_device_kv4_read": (C.c_int, [_P, _SIDP, _SZ, _F32P, _F32P, _F32P, _SZ, C.POINTER(_SZ), _ERR, _SZ]),
    "rs_qwen_device_kv4_evict": (C.c_int, [_P, _SZ, _SIDP, _SZ, _SZ, _SIDP, _ERR, _SZ]),
    "rs_qwen_device_set_capture": (C.c_int, [_P, C.c_int, _ERR, _SZ]),
    "rs_qwen_device_set_profile": (C.c_int, [_P, C.c_int, _ERR, _SZ]),
    "rs_qwen_ep_unique_id": (C.c_int, [C.c_void_p, _SZ, _ERR, _SZ]),
    "rs_qwen_device_ep_init": (C.c_int, [_P, C.c_int, C.c_int, C.c_void_p, _SZ, _SZ, _ERR, _SZ]),
    "rs_qwen_device_ep_window": (C.c_int, [_P, C.c_int, C.c_int, _SZ, C.c_void_p, _SZ, _ERR, _SZ]),
    "rs_qwen_device_ep_connect": (C.c_int, [_P, C.c_void_p, _SZ, _ERR, _SZ]),
    "rs_qwen_device_timing": (C.c_int, [_P, C.POINTER(C.c_double), _SZ, _ERR, _SZ]),
    "rs_qwen_device_debug_routing": (C.c_int, [_P, _I32P, _SZ, _ERR, _SZ]),
    "rs_qwen_device_debug_capture": (C.c_int, [_P, C.c_int, C.c_void_p, _SZ, C.POINTER(_SZ), _ERR, _SZ]),
    "rs_qwen_debug_gemm": (C.c_int, [_P, C.c_int, C.c_int, C.POINTER(C.c_uint16), _SZ, _F32P, _SZ, C.c_int,
                                     C.POINTER(C.c_double), _ERR, _SZ]),
    "rs_qwen_project_noalloc": (C.c_int, [_P, C.c_int, C.c_int, C.c_void_p, _SZ, C.c_void_p, _SZ, C.c_void_p,
                                          _ERR, _SZ]),
    "rs_qwen_kv4_page_bytes": (_SZ, [C.c_int, C.c_int]),
    "rs_qwen_kv4_workspace_bytes": (_SZ, [C.POINTER(Kv4CacheDesc), _SZ, _SZ]),
    "rs_qwen_kv4_append": (C.c_int, [C.POINTER(Kv4CacheDesc), C.POINTER(Kv4AppendArgs), _P, _ERR, _SZ]),
    "rs_qwen_kv4_read": (C.c_int, [C.POINTER(Kv4CacheDesc), _SZ, _P, C.c_uint32, _P, _P, _P, _ERR, _SZ]),
    "rs_qwen_kv4_attention": (C.c_int, [C.POINTER(Kv4CacheDesc), C.POINTER(Kv4AttentionArgs), _P, _ERR, _SZ]),
    "rs_qwen_kv4_evict": (C.c_int, [C.POINTER(Kv4CacheDesc), C.POINTER(Kv4EvictArgs), _P, _ERR, _SZ]),
}

_lib = None


def load(path: Path | None = None):
    """Load libqwen_b200.so; raises if it has not been built (no fallback)."""
    global _lib
    if _lib is None:
        p = Path(path) if path else LIB_PATH
        if not p.exists():
            raise FileNotFoundError(f"{p} missing: build it with python {PKG / 'build.py'}")
        lib = C.CDLL(str(p))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def _errbuf():
    return C.create_string_buffer(1024)


def _call(name, *args):
    e = _errbuf()
    rc = getattr(load(), name)(*args, e, len(e))
    if rc != 0:
        raise NativeError(f"{name}: {e.value.decode(errors='replace')}")


def _ptr(a, t):
    return None if a is None else a.ctypes.data_as(C.POINTER(t))


def config(**kw) -> RsQwenConfig:
    c = RsQwenConfig()
    defaults = dict(activation_precision=1, layer_group=1, validation_mode=0, validation_interval=1,
                    chunk=8, group=64, bits=4, epsilon=1e-6, theta=1e7, interval=4, conv=4)
    defaults.update(kw)
    for k, v in defaults.items():
        setattr(c, k, v)
    return c


def config0(context: int = 512) -> RsQwenConfig:
    """BASELINE configs[0] geometry (tiny hybrid decoder)."""
    return config(hidden=256, layers=4, vocab=4096, q_heads=4, kv_heads=1, head_dim=64, key_heads=2,
                  value_heads=4, key_dim=64, value_dim=64, experts=16, top=2, intermediate=128, shared=128,
                  context=context, rope_dims=16)


def config1(layers: int = 48, context: int = 32768 + 64, vocab: int = 151936) -> RsQwenConfig:
    """BASELINE configs[1] geometry: Qwen3-Next-80B-A3B shapes."""
    return config(hidden=2048, layers=layers, vocab=vocab, q_heads=16, kv_heads=2, head_dim=256, key_heads=16,
                  value_heads=32, key_dim=128, value_dim=128, experts=512, top=10, intermediate=512, shared=512,
                  context=context, rope_dims=64)


def layer_program(cfg: RsQwenConfig):
    arr = (RsQwenLayer * cfg.layers)()
    for i in range(cfg.layers):
        arr[i].index = i
        arr[i].mixer = int((i + 1) % cfg.interval == 0)
    return arr


def state_count(cfg: RsQwenConfig) -> int:
    return load().rs_qwen_state_count(C.byref(cfg))


def ep_unique_id() -> bytes:
    """NCCL unique id (128 bytes) for rs_qwen_device_ep_init, made by rank 0."""
    buf = (C.c_uint8 * 128)()
    _call("rs_qwen_ep_unique_id", buf, 128)
    return bytes(buf)


class WeightStore:
    def __init__(self):
        e = _errbuf()
        self.h = load().rs_mlx_weights_create(e, len(e))
        if not self.h:
            raise NativeError(e.value.decode())

    def synthetic(self, cfg: RsQwenConfig, seed: int, mtp: bool = False):
        self.cfg = cfg
        _call("rs_qwen_weights_synthetic", self.h, C.byref(cfg), seed, int(mtp))
        return self

    def load(self, path):
        """Read one safetensors shard (rs_mlx_weights_load); the device layout is
        built when the first session is created on the store."""
        _call("rs_mlx_weights_load", self.h, str(path).encode())
        return self

    def quant(self, module: str, group: int, bits: int):
        """Per-module quantization override (rs_qwen_quant)."""
        _call("rs_qwen_quant", self.h, module.encode(), group, bits)
        return self

    def forward(self, cfg: RsQwenConfig, tokens, offset: int, old_state=None):
        """rs_qwen_forward: returns (last-row logits [vocab], new_state [state_count])."""
        tok = np.ascontiguousarray(tokens, np.uint32)
        n = state_count(cfg)
        new = np.zeros(n, np.float32)
        old = None if old_state is None else np.ascontiguousarray(old_state, np.float32)
        logits = np.zeros(cfg.vocab, np.float32)
        layers = layer_program(cfg)
        _call("rs_qwen_forward", self.h, 1, C.byref(cfg), layers, cfg.layers, _ptr(tok, C.c_uint32), len(tok),
              offset, _ptr(old, C.c_float), 0 if old is None else old.size, _ptr(new, C.c_float), n,
              _ptr(logits, C.c_float), logits.size, 0, None, 0, None, 0)
        return logits, new

    def weight_bytes(self, name: str, offset: int, count: int, dtype: int = 2) -> bytes:
        buf = (C.c_uint8 * count)()
        _call("rs_mlx_weight_bytes", self.h, name.encode(), None, 0, dtype, offset, buf, count)
        return bytes(buf)

    def close(self):
        if getattr(self, "h", None):
            load().rs_mlx_weights_destroy(self.h)
            self.h = None

    __del__ = close


class DeviceSession:
    """Mirror of QwenDeviceExecutor's native session (src/serving/native_device.rs)."""

    def __init__(self, store: WeightStore, cfg: RsQwenConfig, slots: int, budget_bytes: int):
        self.store, self.cfg = store, cfg
        self.layers = layer_program(cfg)
        e = _errbuf()
        self.h = load().rs_qwen_device_create(store.h, 1, C.byref(cfg), self.layers, cfg.layers, slots,
                                              budget_bytes, e, len(e))
        if not self.h:
            raise NativeError(f"rs_qwen_device_create: {e.value.decode()}")

    def close(self):
        if getattr(self, "h", None):
            load().rs_qwen_device_destroy(self.h)
            self.h = None

    __del__ = close

    def step_ragged(self, parents, positions, counts, tokens, flags=RAGGED_SAMPLED, logits_out=None,
                    sampled_out=None):
        """parents: list of StateId or None. Returns (outs, sampled, logits)."""
        n = len(positions)
        par = (StateId * n)()
        for i, p in enumerate(parents):
            if p is not None:
                par[i] = p
        pos = np.ascontiguousarray(positions, np.uint32)
        cnt = np.ascontiguousarray(counts, np.uint32)
        tok = np.ascontiguousarray(tokens, np.uint32)
        rows = int(cnt.sum()) if flags & RAGGED_ALL_ROWS else n
        outs = (StateId * n)()
        sampled = None
        if flags & RAGGED_SAMPLED:
            sampled = sampled_out if sampled_out is not None else np.zeros(rows, np.uint32)
        logits = None
        if flags & RAGGED_LOGITS:
            logits = logits_out if logits_out is not None else np.zeros((rows, self.cfg.vocab), np.float32)
        _call("rs_qwen_device_step_ragged", self.h, n, par, _ptr(pos, C.c_uint32), _ptr(cnt, C.c_uint32),
              _ptr(tok, C.c_uint32), flags, outs, _ptr(sampled, C.c_uint32), 0 if sampled is None else rows,
              _ptr(logits, C.c_float), 0 if logits is None else logits.size)
        return list(outs), sampled, logits

    def step_ragged_choices(self, parents, positions, counts, tokens, allowed, flags=RAGGED_SAMPLED):
        """step_ragged with constrained greedy selection: allowed[r] is the list of
        legal ids of output row r (empty / None = unconstrained).
        Returns (outs, sampled, logits or None)."""
        n = len(positions)
        par = (StateId * n)()
        for i, p in enumerate(parents):
            if p is not None:
                par[i] = p
        pos = np.ascontiguousarray(positions, np.uint32)
        cnt = np.ascontiguousarray(counts, np.uint32)
        tok = np.ascontiguousarray(tokens, np.uint32)
        rows = int(cnt.sum()) if flags & RAGGED_ALL_ROWS else n
        if len(allowed) != rows:
            raise ValueError("one allowed list per output row")
        lens = [0 if a is None else len(a) for a in allowed]
        offs = np.concatenate([[0], np.cumsum(lens)]).astype(np.uint32)
        ids = np.concatenate([np.asarray(a, np.uint32) for a in allowed if a is not None and len(a)] or
                             [np.zeros(0, np.uint32)]).astype(np.uint32)
        outs = (StateId * n)()
        sampled = np.zeros(rows, np.uint32)
        logits = np.zeros((rows, self.cfg.vocab), np.float32) if flags & RAGGED_LOGITS else None
        _call("rs_qwen_device_step_ragged_choices", self.h, n, par, _ptr(pos, C.c_uint32), _ptr(cnt, C.c_uint32),
              _ptr(tok, C.c_uint32), flags | RAGGED_SAMPLED, _ptr(offs, C.c_uint32),
              _ptr(ids, C.c_uint32) if ids.size else None, ids.size, outs, _ptr(sampled, C.c_uint32), rows,
              _ptr(logits, C.c_float), 0 if logits is None else logits.size)
        return list(outs), sampled, logits

    def decode_batch(self, parents, tokens):
        n = len(parents)
        par = (StateId * n)(*parents)
        tok = np.ascontiguousarray(tokens, np.uint32)
        outs = (StateId * n)()
        logits = np.zeros((n, self.cfg.vocab), np.float32)
        _call("rs_qwen_device_decode_batch", self.h, par, _ptr(tok, C.c_uint32), n, outs,
              _ptr(logits, C.c_float), logits.size)
        return list(outs), logits

    def step(self, previous, position, tokens, block=False, hidden=False):
        tok = np.ascontiguousarray(tokens, np.uint32)
        out = StateId()
        rows = len(tok) if block else 1
        logits = np.zeros((rows, self.cfg.vocab), np.float32)
        prev = C.byref(previous) if previous is not None else None
        name = {(False, False): "rs_qwen_device_step", (True, False): "rs_qwen_device_block",
                (False, True): "rs_qwen_device_hidden_step", (True, True): "rs_qwen_device_hidden_block"}[(block, hidden)]
        if name == "rs_qwen_device_step":
            _call(name, self.h, prev, position, _ptr(tok, C.c_uint32), len(tok), C.byref(out),
                  _ptr(logits, C.c_float), logits.size, None, 0)
        else:
            _call(name, self.h, prev, position, _ptr(tok, C.c_uint32), len(tok), C.byref(out),
                  _ptr(logits, C.c_float), logits.size)
        return out, logits

    def step_sampled(self, previous, position, tokens):
        tok = np.ascontiguousarray(tokens, np.uint32)
        out, token = StateId(), C.c_uint32()
        prev = C.byref(previous) if previous is not None else None
        _call("rs_qwen_device_step_sampled", self.h, prev, position, _ptr(tok, C.c_uint32), len(tok),
              C.byref(out), C.byref(token))
        return out, token.value

    def release(self, sid: StateId):
        _call("rs_qwen_device_release", self.h, C.byref(sid))

    def verify_accept(self, parents, seeds, drafts, eos=(), flags=0, width=None):
        """Speculative verify + accept (rs_qwen_device_mtp_verify_accept).
        drafts: list of per-sequence draft lists. Returns (outs, accepted, emitted lists)."""
        n = len(parents)
        width = max([len(x) for x in drafts] + [0]) if width is None else width
        par = (StateId * n)(*parents)
        seed = np.ascontiguousarray(seeds, np.uint32)
        nd = np.array([len(x) for x in drafts], np.uint32)
        dr = np.zeros((n, max(width, 1)), np.uint32)
        for i, x in enumerate(drafts):
            dr[i, :len(x)] = x
        eo = np.ascontiguousarray(eos, np.uint32)
        outs = (StateId * n)()
        acc = np.zeros(n, np.uint32)
        em = np.zeros((n, width + 1), np.uint32)
        ne = np.zeros(n, np.uint32)
        _call("rs_qwen_device_mtp_verify_accept", self.h, n, par, _ptr(seed, C.c_uint32), _ptr(dr, C.c_uint32),
              _ptr(nd, C.c_uint32), width, _ptr(eo, C.c_uint32) if len(eo) else None, len(eo), flags, outs,
              _ptr(acc, C.c_uint32), _ptr(em, C.c_uint32), _ptr(ne, C.c_uint32))
        return list(outs), [int(a) for a in acc], [list(map(int, em[i, :ne[i]])) for i in range(n)]

    def snapshot(self, sid: StateId):
        n = state_count(self.cfg)
        out = np.zeros(n, np.float32)
        _call("rs_qwen_device_snapshot", self.h, C.byref(sid), _ptr(out, C.c_float), n)
        return out

    def hidden_snapshot(self, sid: StateId, rows: int):
        out = np.zeros((rows, self.cfg.hidden), np.float32)
        _call("rs_qwen_device_hidden_snapshot", self.h, C.byref(sid), _ptr(out, C.c_float), out.size)
        return out

    def stats(self):
        out = (C.c_uint64 * STATS_COUNT)()
        _call("rs_qwen_device_stats", self.h, out, STATS_COUNT)
        return list(out)

    def drain(self) -> int:
        n = C.c_uint64()
        _call("rs_qwen_device_drain", self.h, C.byref(n))
        return n.value

    def mtp_attach(self, store):
        _call("rs_qwen_device_mtp_attach", self.h, store.h)

    def mtp_step(self, previous, source, tokens, row: int = 0, draft_source: int = 0):
        """One MTP draft step (rs_qwen_device_mtp_step); returns (draft version, last-row logits)."""
        tok = np.ascontiguousarray(tokens, np.uint32)
        out = StateId()
        logits = np.zeros(self.cfg.vocab, np.float32)
        _call("rs_qwen_device_mtp_step", self.h, None if previous is None else C.byref(previous), C.byref(source),
              draft_source, row, _ptr(tok, C.c_uint32), len(tok), C.byref(out), _ptr(logits, C.c_float),
              logits.size, 0)
        return out, logits

    def mtp_release(self, sid: StateId):
        _call("rs_qwen_device_mtp_release", self.h, C.byref(sid))

    def mtp_snapshot(self, sid: StateId, rows: int):
        """(K [kv, context, d], V [kv, context, d], hidden [rows, hidden]) of a draft version."""
        c = self.cfg
        per = c.kv_heads * c.context * c.head_dim
        out = np.zeros(2 * per + rows * c.hidden, np.float32)
        _call("rs_qwen_device_mtp_snapshot", self.h, C.byref(sid), _ptr(out, C.c_float), out.size)
        kv = out[:2 * per].reshape(2, c.kv_heads, c.context, c.head_dim)
        return kv[0], kv[1], out[2 * per:].reshape(rows, c.hidden)

    def synthetic_state(self, position: int, seed: int) -> StateId:
        out = StateId()
        _call("rs_qwen_device_synthetic_state", self.h, position, seed, C.byref(out))
        return out

    def kv4(self, track: bool = False):
        """Attention pages in 4 bits (rs_qwen_device_kv4); before any admission and mtp_attach."""
        _call("rs_qwen_device_kv4", self.h, int(track))
        return self

    def kv4_read(self, sid: StateId, layer: int, weights: bool = False):
        """Keys, values [kv_heads, held, head_dim] and weights [kv_heads, held] (or None) that a version's cache
        holds in attention layer `layer` (rs_qwen_device_kv4_read)."""
        held = C.c_size_t()
        _call("rs_qwen_device_kv4_read", self.h, C.byref(sid), layer, None, None, None, 0, C.byref(held))
        shape = (self.cfg.kv_heads, held.value, self.cfg.head_dim)
        k, v = np.zeros(shape, np.float32), np.zeros(shape, np.float32)
        w = np.zeros(shape[:2], np.float32) if weights else None
        _call("rs_qwen_device_kv4_read", self.h, C.byref(sid), layer, _ptr(k, C.c_float), _ptr(v, C.c_float),
              _ptr(w, C.c_float), held.value, C.byref(held))
        return k, v, w

    def kv4_evict(self, sids, keep: int, recent: int):
        """New versions that keep `keep` keys per layer and KV head (rs_qwen_device_kv4_evict)."""
        n = len(sids)
        ids, outs = (StateId * n)(*sids), (StateId * n)()
        _call("rs_qwen_device_kv4_evict", self.h, n, ids, keep, recent, outs)
        return list(outs)

    def set_capture(self, routing: bool):
        _call("rs_qwen_device_set_capture", self.h, int(routing))

    def ep_init(self, world: int, rank: int, uid: bytes, cap_tokens: int):
        """Join the expert-parallel group (see rs_qwen_device_ep_init)."""
        buf = (C.c_uint8 * len(uid)).from_buffer_copy(uid)
        _call("rs_qwen_device_ep_init", self.h, world, rank, buf, len(uid), cap_tokens)

    def ep_window(self, world: int, rank: int, cap_tokens: int) -> bytes:
        """Expert parallelism over direct NVLink stores, step 1: allocate this
        rank's window; returns its CUDA IPC handle (64 bytes) for the peers."""
        buf = (C.c_uint8 * 64)()
        _call("rs_qwen_device_ep_window", self.h, world, rank, cap_tokens, buf, 64)
        return bytes(buf)

    def ep_connect(self, handles):
        """Step 2: every rank's window handle, in rank order."""
        blob = b"".join(handles)
        buf = (C.c_uint8 * len(blob)).from_buffer_copy(blob)
        _call("rs_qwen_device_ep_connect", self.h, buf, len(blob))

    def set_profile(self, on: bool):
        _call("rs_qwen_device_set_profile", self.h, int(on))

    def timing(self):
        """(last step device ms, cumulative device ms, timed steps, per-stage ms[19])."""
        out = (C.c_double * 22)()
        _call("rs_qwen_device_timing", self.h, out, 22)
        return out[0], out[1], int(out[2]), list(out[3:])

    def debug_gemm(self, which: int, layer: int, x_f16, rows: int, engine: int = 0):
        """Run one dense GEMM (0 in_proj, 1 out_proj, 2 router, 3 lm_head) on IEEE-half
        input bits [T][k]; returns (y, ms)."""
        x = np.ascontiguousarray(x_f16, np.uint16)
        T = x.shape[0]
        y = np.zeros((T, rows), np.float32)
        ms = C.c_double()
        _call("rs_qwen_debug_gemm", self.h, which, layer, x.ctypes.data_as(C.POINTER(C.c_uint16)), T,
              _ptr(y, C.c_float), y.size, engine, C.byref(ms))
        return y, ms.value

    def project_noalloc(self, which: int, layer: int, x_device_ptr: int, T: int, y_device_ptr: int, y_count: int,
                        stream_ptr: int = 0):
        """Allocation-free dense projection on device buffers (rs_qwen_project_noalloc):
        y (fp32 [T][rows]) = x (IEEE half [T][k]) . W; raises on error, including T x rows
        beyond the 16 MiB static scratch."""
        _call("rs_qwen_project_noalloc", self.h, which, layer, C.c_void_p(x_device_ptr), T,
              C.c_void_p(y_device_ptr), y_count, C.c_void_p(stream_ptr or None))

    def debug_capture(self, what: int, dtype=np.int32, capacity: int = 1 << 26):
        """Raw last-step intermediates (see rs_qwen_device_debug_capture)."""
        buf = np.zeros(capacity // np.dtype(dtype).itemsize, dtype)
        n = C.c_size_t()
        _call("rs_qwen_device_debug_capture", self.h, what, buf.ctypes.data_as(C.c_void_p), buf.nbytes, C.byref(n))
        return buf[: n.value // np.dtype(dtype).itemsize].copy()

    def debug_routing(self, tokens: int):
        out = np.zeros((self.cfg.layers, tokens, self.cfg.top), np.int32)
        _call("rs_qwen_device_debug_routing", self.h, _ptr(out, C.c_int32), out.size)
        return out


# ---- 4-bit paged KV cache ----

KV4_PAGE = 16  # tokens per page
# the argument structs, packed in one call
_KV4_APPEND = struct.Struct("=" + 3 * "Qqq" + "IIQQQQQQffii")
_KV4_ATTENTION = struct.Struct("=" + 3 * "Qqq" + "IIQQQQQQqf4xQQQqQQ")
_KV4_EVICT = struct.Struct("=QQQqQqQqiiQQQq")


def _pack(kind, layout, *values):
    try:
        return kind.from_buffer_copy(layout.pack(*values))
    except (struct.error, OverflowError) as e:
        raise ValueError(f"kv4: argument out of range: {e}") from None


assert _KV4_APPEND.size == C.sizeof(Kv4AppendArgs) and _KV4_ATTENTION.size == C.sizeof(Kv4AttentionArgs)
assert _KV4_EVICT.size == C.sizeof(Kv4EvictArgs)


def kv4_page_bytes(kv_heads: int, head_dim: int) -> int:
    """Pool bytes of one 16-token page (rs_qwen_kv4_page_bytes)."""
    n = load().rs_qwen_kv4_page_bytes(kv_heads, head_dim)
    if not n:
        raise NativeError("kv4: head_dim must be 64, 128 or 256 and kv_heads 1 to 1024")
    return n


class Kv4Cache:
    """4-bit paged KV cache of one attention layer (rs_qwen_kv4_*) on CUDA tensors.

    `pool` is a contiguous uint8 tensor holding whole pages (kv4_page_bytes each);
    it stays the caller's. Every other argument is a tensor on the pool's device.
    Calls enqueue on `stream` (a torch stream or raw handle; default: the current
    stream of that device) and do not synchronise; a tensor that belongs to
    another stream must be kept alive and ordered by the caller, as for any
    kernel. `status`, a one-element int32 tensor, receives bit 2 when a kernel
    met a page id, slot or length out of range (see check())."""

    def __init__(self, pool, q_heads: int, kv_heads: int, head_dim: int, status=None):
        import torch
        self._current_stream = torch.cuda.current_stream
        self._synchronize = torch.cuda.synchronize
        self._f32, self._i32, self._i64, self._u8 = torch.float32, torch.int32, torch.int64, torch.uint8
        self._types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        page = kv4_page_bytes(kv_heads, head_dim)
        if pool.dtype != torch.uint8 or not pool.is_contiguous() or not pool.is_cuda:
            raise ValueError("kv4: the pool is a contiguous uint8 CUDA tensor")
        if pool.numel() < page or pool.numel() % page:
            raise ValueError(f"kv4: the pool holds whole pages of {page} bytes")
        if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or
                                   status.device != pool.device):
            raise ValueError("kv4: status is one int32 on the pool's device")
        self.pool, self.status, self.device = pool, status, pool.device
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.pages, self._index = pool.numel() // page, pool.get_device()
        self.desc = Kv4CacheDesc(pool.device.index, q_heads, kv_heads, head_dim, self.pages, pool.data_ptr(),
                                 None if status is None else status.data_ptr())
        self._ref = C.byref(self.desc)
        if not load().rs_qwen_kv4_workspace_bytes(self._ref, 1, 1):
            raise NativeError("kv4: q_heads must be 1 to 16 times kv_heads")

    def _stream(self, stream):
        if stream is None:
            return self._current_stream(self._index).cuda_stream
        return getattr(stream, "cuda_stream", stream)

    # The checks below run on every call: a decode step's kernels take less time than
    # a few microseconds of them. Arguments are packed in the C struct's layout
    # (ctypes sets fields one by one, three times as slow); a null pointer is 0.

    def _rows(self, x, name, tokens, heads, dtype=None):
        if x is None:
            return 0, 0, 0
        if x.shape != (tokens, heads, self.head_dim) or x.get_device() != self._index:
            raise ValueError(f"kv4: {name} must be [{tokens}, {heads}, {self.head_dim}] on {self.device}")
        if dtype is not None and x.dtype != dtype:
            raise ValueError(f"kv4: {name} must be {dtype}")
        s = x.stride()
        if s[2] != 1 and x.numel():
            raise ValueError(f"kv4: the last dimension of {name} must be contiguous")
        return x.data_ptr(), s[0], s[1]

    def _array(self, x, name, dtype, shape=None, optional=False):
        """Pointer of a contiguous array."""
        if x is None:
            if optional:
                return 0
            raise ValueError(f"kv4: {name} is missing")
        if x.dtype != dtype or x.get_device() != self._index or not x.is_contiguous():
            raise ValueError(f"kv4: {name} must be a contiguous {dtype} tensor on {self.device}")
        if shape is not None and x.shape != shape:
            raise ValueError(f"kv4: {name} must be of shape {list(shape)}")
        return x.data_ptr()

    def _type(self, x, name):
        code = self._types.get(x.dtype)
        if code is None:
            raise ValueError(f"kv4: {name} must be float32, float16 or bfloat16")
        return code

    def workspace_bytes(self, n_seq: int, tokens: int) -> int:
        """Workspace of attention() for up to this many sequences and query tokens."""
        return load().rs_qwen_kv4_workspace_bytes(self._ref, n_seq, tokens)

    def append(self, q, k, v, positions, slots, q_out, q_norm=None, k_norm=None, epsilon: float = 1e-6,
               theta: float = 1e7, rope_dims: int = 0, stream=None):
        """Norm, rotation and 4-bit write of new tokens (rs_qwen_kv4_append). q [T, q_heads, D], k and v
        [T, kv_heads, D] of one dtype, any token / head strides; q (with q_out) or k and v may be None."""
        x = q if q is not None else k
        if x is None or (k is None) != (v is None) or (q is None) != (q_out is None):
            raise ValueError("kv4: append takes q with q_out, k with v, or all four")
        T, D, one, dtype = x.shape[0], self.head_dim, self._f32, x.dtype
        args = _pack(
            Kv4AppendArgs, _KV4_APPEND, *self._rows(q, "q", T, self.q_heads, dtype), *self._rows(k, "k", T, self.kv_heads, dtype),
            *self._rows(v, "v", T, self.kv_heads, dtype), self._type(x, "q"),
            0 if q_out is None else self._type(q_out, "q_out"), T,
            self._array(q_norm, "q_norm", one, (D,), True), self._array(k_norm, "k_norm", one, (D,), True),
            self._array(positions, "positions", self._i32, (T,), rope_dims == 0),
            self._array(slots, "slots", self._i64, (T,), k is None),
            0 if q_out is None else self._array(q_out, "q_out", q_out.dtype, (T, self.q_heads, D)),
            epsilon, theta, rope_dims, 0)
        _call("rs_qwen_kv4_append", self._ref, C.byref(args), self._stream(stream))

    def read(self, slots, k, v, stream=None):
        """Cached tokens back as values (rs_qwen_kv4_read): k, v [len(slots), kv_heads, D]."""
        shape = (slots.shape[0], self.kv_heads, self.head_dim)
        _call("rs_qwen_kv4_read", self._ref, shape[0], self._array(slots, "slots", self._i64, shape[:1]),
              self._type(k, "k"), self._array(k, "k", k.dtype, shape), self._array(v, "v", k.dtype, shape),
              self._stream(stream))

    def attention(self, q, cu_seqlens, kv_lens, block_table, out, workspace, max_count: int, gate=None, lse=None,
                  weights_in=None, weights_out=None, scale: float = 0.0, stream=None):
        """Ragged causal attention over the pages (rs_qwen_kv4_attention). block_table: int32 [n_seq, pages];
        weights_in / weights_out: float32 [n_seq, kv_heads, columns]; workspace: uint8, workspace_bytes()."""
        if q.dim() != 3 or block_table.dim() != 2:
            raise ValueError("kv4: q must be [T, q_heads, head_dim] and block_table [n_seq, pages]")
        if gate is not None and gate.dtype != self._f32:
            raise ValueError("kv4: the gate must be float32")
        T, n, pages, one, whole = q.shape[0], kv_lens.shape[0], block_table.shape[1], self._f32, self._i32
        columns = 0
        if weights_out is not None:
            columns = weights_out.shape[-1]
        elif weights_in is not None:
            raise ValueError("kv4: weights_in needs weights_out")
        wshape = (n, self.kv_heads, columns)
        args = _pack(
            Kv4AttentionArgs, _KV4_ATTENTION, *self._rows(q, "q", T, self.q_heads), *self._rows(gate, "gate", T, self.q_heads),
            *self._rows(out, "out", T, self.q_heads, q.dtype), self._type(q, "q"), 0, n, T, max_count,
            self._array(cu_seqlens, "cu_seqlens", whole, (n + 1,)), self._array(kv_lens, "kv_lens", whole, (n,)),
            self._array(block_table, "block_table", whole, (n, pages)), pages, scale,
            self._array(lse, "lse", one, (T, self.q_heads), True),
            self._array(weights_in, "weights_in", one, wshape, True),
            self._array(weights_out, "weights_out", one, wshape, True), columns,
            self._array(workspace, "workspace", self._u8), workspace.numel())
        _call("rs_qwen_kv4_attention", self._ref, C.byref(args), self._stream(stream))

    def evict(self, kv_lens, src_table, dst_table, weights, keep: int, recent: int, kept, new_lens, weights_out=None,
              stream=None):
        """Keeps the most attended keys of every sequence and KV head (rs_qwen_kv4_evict); the kept keys move to
        the pages of dst_table."""
        n, one, whole = kv_lens.shape[0], self._f32, self._i32
        args = _pack(
            Kv4EvictArgs, _KV4_EVICT, n, self._array(kv_lens, "kv_lens", whole, (n,)),
            self._array(src_table, "src_table", whole, (n, src_table.shape[1])), src_table.shape[1],
            self._array(dst_table, "dst_table", whole, (n, dst_table.shape[1])), dst_table.shape[1],
            self._array(weights, "weights", one, (n, self.kv_heads, weights.shape[-1])), weights.shape[-1], keep, recent,
            self._array(kept, "kept", whole, (n, self.kv_heads, keep)), self._array(new_lens, "new_lens", whole, (n,)),
            self._array(weights_out, "weights_out", one,
                        None if weights_out is None else (n, self.kv_heads, weights_out.shape[-1]), True),
            0 if weights_out is None else weights_out.shape[-1])
        _call("rs_qwen_kv4_evict", self._ref, C.byref(args), self._stream(stream))

    def check(self):
        """Reads and clears the status word; raises if a kernel met an index out of range. Waits for the whole device:
        calls may have been made on any of its streams."""
        if self.status is not None:
            self._synchronize(self.device)
            bits = int(self.status.item())
            if bits:
                self.status.zero_()
                raise NativeError(f"kv4: device error flag {bits}")
