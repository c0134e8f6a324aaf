"""ctypes binding of libffn_b200.so for Python callers (tests, bench, smoke).

The library's C-ABI (include/ffn_b200.h, include/merkaba_hw_addon.h) is the
product; this module only marshals torch CUDA tensors into it.  PyTorch here
is plumbing: device memory, streams and torch.distributed.  There is no Python
or CPU compute path: every function below runs a CUDA kernel of the library,
and using it without the built library raises.
"""
from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "_build", "libffn_b200.so")

FMT_NVFP4, FMT_TERNARY, FMT_MXFP4, FMT_MXFP8 = 0, 1, 2, 3
SCORE_REF, SCORE_SIGMOID = 0, 1
ROUTER_EXACT, ROUTER_TENSOR = 0, 1
PATH_AUTO, PATH_GEMV, PATH_GROUPED, PATH_FP4 = 0, 1, 2, 3
GROUPED_MIN_PAIRS = 48
DT_F32, DT_BF16, DT_F16 = 0, 1, 2
ACT_NONE, ACT_SWIGLU = 0, 1
GATE_NONE, GATE_CHANNEL, GATE_TOKEN = 0, 1, 2
ERRORS = {0: "OK", -1: "EINVAL", -2: "ECUDA", -3: "ENOSPC", -4: "ENCCL", -5: "EUNSUP"}

# Symbols the public headers declare (checked by the CPU test suite).
EXPORTS = [
    "merkaba_hardware_addon_v1",
    "gx10_rust_nvfp4_mlp_accum", "gx10_rust_ternary_158_mlp_accum",
    "gx10_rust_nvfp4_mlp_batch", "gx10_rust_ternary_158_mlp_batch",
    "gx10_rust_register_shard_bounds", "gx10_rust_register_host_range",
    "ffn_b200_version", "ffn_b200_last_error", "ffn_b200_launch_count", "ffn_b200_set_device",
    "ffn_b200_matvec_ws_bytes", "ffn_b200_nvfp4_matvec", "ffn_b200_ternary_matvec",
    "ffn_b200_expert_ws_bytes", "ffn_b200_expert_forward", "ffn_b200_expert_forward_noalloc",
    "ffn_b200_moe_ws_bytes", "ffn_b200_moe_layer",
    "ffn_b200_key", "ffn_b200_gen_nvfp4", "ffn_b200_gen_ternary", "ffn_b200_gen_core",
    "ffn_b200_gen_normal", "ffn_b200_dequant_nvfp4", "ffn_b200_dequant_ternary",
    "ffn_b200_set_batch_input", "ffn_b200_release_host_ranges", "ffn_b200_host_cache_bytes",
    "ffn_b200_profile_enable", "ffn_b200_profile_kinds", "ffn_b200_profile_read",
    "ffn_b200_ep_handle_bytes", "ffn_b200_ep_create", "ffn_b200_ep_connect", "ffn_b200_ep_part",
    "ffn_b200_ep_allreduce", "ffn_b200_ep_error", "ffn_b200_ep_destroy",
    "ffn_b200_mxfp4_matvec", "gx10_rust_mxfp4_matvec", "gx10_rust_mxfp4_mlp_accum",
    "ffn_b200_mxfp8_matvec", "gx10_rust_mxfp8_mlp_accum", "gx10_rust_mxfp8_mlp_batch",
    "ffn_b200_st_open", "ffn_b200_st_close", "ffn_b200_st_count", "ffn_b200_st_name",
    "ffn_b200_st_find", "ffn_b200_st_expert_bytes", "ffn_b200_st_load_expert",
    "ffn_b200_compress_ws_bytes", "ffn_b200_compress_ternary_b64",
    "ffn_b200_quantize_nvfp4x4", "ffn_b200_ep_moe_layer", "ffn_b200_set_host_cache_budget",
    "ffn_b200_topk", "ffn_b200_quantize_nvfp4_terms", "ffn_b200_fp4_pack_bytes",
    "ffn_b200_pack_nvfp4_expert",
    "ffn_b200_quantize_int8", "ffn_b200_int8_matmul", "ffn_b200_int8_linear_ws_bytes",
    "ffn_b200_int8_linear",
    "ffn_b200_moe_sort", "ffn_b200_moe_permute", "ffn_b200_moe_combine", "ffn_b200_moe_combine_bwd",
    "ffn_b200_block_norm", "ffn_b200_block_norm_bwd_ws_bytes", "ffn_b200_block_norm_bwd",
]

# Kernel kinds of ffn_b200_profile_read (FFN_B200_K_*).
K_XPREP, K_ROUTER, K_TOPK, K_GROUP, K_GATEUP_NVFP4, K_DOWN_NVFP4 = 0, 1, 2, 3, 4, 5
K_GATEUP_TERNARY, K_DOWN_TERNARY, K_COREZ, K_COMBINE, K_MATVEC, K_OTHER = 6, 7, 8, 9, 10, 11
K_GEMM_GATEUP, K_GEMM_DOWN, K_QUANT, K_FP4_GATEUP, K_FP4_DOWN = 12, 13, 14, 15, 16
K_ROUTE, K_NORM, K_INT8_QUANT, K_INT8_GEMM = 17, 18, 19, 20
K_NAMES = ["xprep", "router", "topk", "group", "gateup_nvfp4", "down_nvfp4", "gateup_ternary",
           "down_ternary", "corez", "combine", "matvec", "other", "gemm_gateup", "gemm_down",
           "quant", "fp4_gateup", "fp4_down", "route", "norm", "int8_quant", "int8_gemm"]


def build() -> str:
    subprocess.run(["make", "-s", "-C", HERE, "-j8", f"PYTHON={sys.executable}"], check=True)
    return LIB_PATH


class FfnError(RuntimeError):
    pass


# ------------------------------------------------------------ C structs
class NvMat(C.Structure):
    _fields_ = [("w", C.c_void_p), ("s", C.c_void_p), ("gs", C.c_float),
                ("reserved", C.c_uint32)]


class TnMat(C.Structure):
    _fields_ = [("p", C.c_void_p), ("rs", C.c_void_p), ("core_a", C.c_void_p),
                ("core_a_sc", C.c_void_p), ("core_b", C.c_void_p), ("core_b_sc", C.c_void_p),
                ("bs", C.c_void_p)]


class Expert(C.Structure):
    _fields_ = [("format", C.c_int32), ("proj_scale", C.c_float), ("nv", NvMat * 3),
                ("tn", TnMat * 3), ("fp4_gu", C.c_void_p), ("fp4_dn", C.c_void_p)]


class MoeDesc(C.Structure):
    _fields_ = [("hidden", C.c_size_t), ("inter", C.c_size_t), ("n_experts", C.c_size_t),
                ("top_k", C.c_size_t), ("experts", C.c_void_p), ("router_w", C.c_void_p),
                ("router_bias", C.c_void_p), ("score_fn", C.c_int32),
                ("router_mode", C.c_int32), ("expert_begin", C.c_int32),
                ("expert_end", C.c_int32), ("has_nvfp4", C.c_int32),
                ("has_ternary", C.c_int32), ("norm_w", C.c_void_p), ("norm_eps", C.c_float),
                ("path", C.c_int32), ("has_mxfp4", C.c_int32), ("fp4_packed", C.c_int32)]


class BlockNormDesc(C.Structure):
    _fields_ = [("rows", C.c_size_t), ("cols", C.c_size_t), ("dtype", C.c_int32),
                ("gate_kind", C.c_int32), ("post_w", C.c_void_p), ("gate", C.c_void_p),
                ("pre_w", C.c_void_p), ("alpha", C.c_float), ("beta", C.c_float),
                ("eps", C.c_float), ("reserved", C.c_uint32)]


assert C.sizeof(Expert) == 264, C.sizeof(Expert)

_lib = None


def lib() -> C.CDLL:
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FfnError(f"{LIB_PATH} is missing: build it with `make -C {HERE}` "
                           "(or __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        sz, vp, f32, i32, u64 = C.c_size_t, C.c_void_p, C.c_float, C.c_int, C.c_uint64
        L.ffn_b200_version.restype = C.c_char_p
        L.ffn_b200_last_error.restype = C.c_char_p
        L.ffn_b200_launch_count.restype = u64
        L.ffn_b200_set_device.argtypes = [i32]
        L.ffn_b200_matvec_ws_bytes.restype = sz
        L.ffn_b200_matvec_ws_bytes.argtypes = [sz, sz]
        L.ffn_b200_nvfp4_matvec.argtypes = [sz, sz, sz, C.POINTER(NvMat), vp, vp, vp, sz, vp]
        L.ffn_b200_ternary_matvec.argtypes = [sz, sz, sz, C.POINTER(TnMat), vp, vp, vp, sz, vp]
        L.ffn_b200_mxfp4_matvec.argtypes = [sz, sz, sz, C.POINTER(NvMat), vp, vp, vp, sz, vp]
        L.ffn_b200_quantize_nvfp4x4.argtypes = [sz, sz, vp, sz, vp, vp, vp, vp]
        L.ffn_b200_topk.argtypes = [sz, sz, sz, C.c_int32, vp, sz, vp, vp, vp, vp]
        L.ffn_b200_quantize_nvfp4_terms.argtypes = [sz, sz, sz, vp, sz, vp, vp, vp, vp]
        L.ffn_b200_fp4_pack_bytes.restype = sz
        L.ffn_b200_fp4_pack_bytes.argtypes = [sz, sz, C.c_int]
        L.ffn_b200_pack_nvfp4_expert.argtypes = [sz, sz, C.POINTER(Expert), vp, vp, vp]
        L.gx10_rust_mxfp4_matvec.argtypes = [sz, sz, vp, vp, vp, vp]
        L.gx10_rust_mxfp4_matvec.restype = C.c_bool
        L.gx10_rust_mxfp4_mlp_accum.argtypes = [sz, sz, vp, vp, vp, vp, vp, vp, vp, vp, f32,
                                                C.c_bool, C.c_bool]
        L.gx10_rust_mxfp4_mlp_accum.restype = C.c_bool
        L.ffn_b200_mxfp8_matvec.argtypes = [sz, sz, sz, C.POINTER(NvMat), vp, vp, vp, sz, vp]
        L.gx10_rust_mxfp8_mlp_accum.argtypes = [sz, sz, vp, vp, vp, vp, vp, vp, vp, vp, f32,
                                                C.c_bool, C.c_bool]
        L.gx10_rust_mxfp8_mlp_accum.restype = C.c_bool
        L.gx10_rust_mxfp8_mlp_batch.argtypes = [sz, sz, sz, vp, vp, vp, vp, vp, vp, vp, sz, vp,
                                                C.c_bool]
        L.gx10_rust_mxfp8_mlp_batch.restype = C.c_bool
        L.gx10_rust_nvfp4_mlp_accum.argtypes = [sz, sz, vp, vp, f32, vp, vp, f32, vp, vp, f32, vp,
                                                vp, f32, C.c_bool, C.c_bool]
        L.gx10_rust_nvfp4_mlp_accum.restype = C.c_bool
        L.gx10_rust_ternary_158_mlp_accum.argtypes = [sz, sz, vp, vp, vp, vp, vp, vp, f32, vp, vp,
                                                      f32, C.c_bool, C.c_bool]
        L.gx10_rust_ternary_158_mlp_accum.restype = C.c_bool
        L.gx10_rust_nvfp4_mlp_batch.argtypes = [sz, sz, sz, vp, vp, f32, vp, vp, f32, vp, vp, f32,
                                                sz, vp, vp, sz, vp, C.c_bool]
        L.gx10_rust_nvfp4_mlp_batch.restype = C.c_bool
        L.gx10_rust_ternary_158_mlp_batch.argtypes = [sz, sz, sz, vp, vp, vp, vp, vp, vp, f32, sz,
                                                      vp, vp, sz, vp, C.c_bool]
        L.gx10_rust_ternary_158_mlp_batch.restype = C.c_bool
        L.ffn_b200_compress_ws_bytes.restype = sz
        L.ffn_b200_compress_ws_bytes.argtypes = [sz, sz]
        L.ffn_b200_compress_ternary_b64.argtypes = [sz, sz, vp, vp, f32, u64, vp, vp, vp, vp, vp, vp,
                                                    vp, vp, sz, vp]
        L.ffn_b200_expert_ws_bytes.restype = sz
        L.ffn_b200_expert_ws_bytes.argtypes = [sz, sz, sz]
        L.ffn_b200_expert_forward.argtypes = [sz, sz, sz, C.POINTER(Expert), vp, vp, f32, i32,
                                              vp, sz, vp]
        L.ffn_b200_expert_forward_noalloc.argtypes = [sz, sz, sz, C.POINTER(Expert), vp, vp, f32,
                                                      i32, vp]
        L.ffn_b200_moe_ws_bytes.restype = sz
        L.ffn_b200_moe_ws_bytes.argtypes = [C.POINTER(MoeDesc), sz]
        L.ffn_b200_moe_layer.argtypes = [C.POINTER(MoeDesc), sz, vp, vp, vp, vp, vp, vp, sz, vp]
        L.ffn_b200_key.restype = u64
        L.ffn_b200_key.argtypes = [u64, u64]
        L.ffn_b200_gen_nvfp4.argtypes = [u64, sz, sz, vp, vp, vp]
        L.ffn_b200_gen_ternary.argtypes = [u64, sz, sz, vp, vp, vp]
        L.ffn_b200_gen_core.argtypes = [u64, sz, sz, vp, vp, vp, vp, vp]
        L.ffn_b200_gen_normal.argtypes = [u64, sz, f32, vp, vp]
        L.ffn_b200_dequant_nvfp4.argtypes = [sz, sz, vp, vp, vp, vp]
        L.ffn_b200_dequant_ternary.argtypes = [sz, sz, vp, vp, vp]
        L.ffn_b200_set_batch_input.argtypes = [vp, sz, sz]
        L.ffn_b200_host_cache_bytes.restype = sz
        L.ffn_b200_set_host_cache_budget.argtypes = [sz]
        L.merkaba_hardware_addon_v1.restype = vp
        L.ffn_b200_profile_enable.argtypes = [i32]
        L.ffn_b200_profile_kinds.argtypes = [C.c_uint32]
        L.ffn_b200_ep_handle_bytes.restype = sz
        L.ffn_b200_ep_create.argtypes = [i32, i32, sz, sz, vp, C.POINTER(vp)]
        L.ffn_b200_ep_connect.argtypes = [vp, vp]
        L.ffn_b200_ep_part.argtypes = [vp]
        L.ffn_b200_ep_part.restype = vp
        L.ffn_b200_ep_allreduce.argtypes = [vp, sz, vp, vp, vp]
        L.ffn_b200_ep_moe_layer.argtypes = [vp, C.POINTER(MoeDesc), sz, vp, vp, vp, vp, vp, vp, sz, vp]
        L.ffn_b200_ep_error.argtypes = [vp, C.POINTER(C.c_int)]
        L.ffn_b200_ep_destroy.argtypes = [vp]
        L.ffn_b200_profile_read.argtypes = [i32, C.POINTER(C.c_double), C.POINTER(C.c_uint64)]
        L.ffn_b200_quantize_int8.argtypes = [sz, sz, C.c_int32, vp, sz, C.c_int32, vp, vp, sz, vp, vp]
        L.ffn_b200_int8_matmul.argtypes = [sz, sz, sz, sz, vp, vp, sz, vp, vp, sz, vp, vp, C.c_int32,
                                           vp, sz, vp]
        L.ffn_b200_int8_linear_ws_bytes.restype = sz
        L.ffn_b200_int8_linear_ws_bytes.argtypes = [sz, sz, sz, vp]
        L.ffn_b200_int8_linear.argtypes = [sz, sz, sz, sz, vp, C.c_int32, vp, sz, vp, sz, vp, vp, C.c_int32,
                                           vp, sz, vp, sz, vp]
        L.ffn_b200_moe_sort.argtypes = [sz, sz, vp, C.c_int32, C.c_int32, vp, vp, vp, vp]
        L.ffn_b200_moe_permute.argtypes = [sz, sz, sz, vp, sz, vp, sz, vp, sz, vp, vp, vp]
        L.ffn_b200_moe_combine.argtypes = [sz, sz, sz, C.c_int32, vp, sz, sz, vp, vp, vp, sz, vp, sz,
                                           vp]
        L.ffn_b200_moe_combine_bwd.argtypes = [sz, sz, sz, C.c_int32, vp, sz, vp, sz, sz, vp, vp, vp,
                                               sz, vp, vp]
        pd = C.POINTER(BlockNormDesc)
        L.ffn_b200_block_norm.argtypes = [pd, vp, sz, vp, sz, vp, sz, vp, sz, vp, sz, vp, vp]
        L.ffn_b200_block_norm_bwd_ws_bytes.restype = sz
        L.ffn_b200_block_norm_bwd_ws_bytes.argtypes = [pd]
        L.ffn_b200_block_norm_bwd.argtypes = [pd, vp, sz, vp, sz, vp, sz, vp, sz, vp, sz, vp, sz, vp,
                                              vp, vp, vp, sz, vp]
        L.ffn_b200_st_open.argtypes = [C.c_char_p, C.POINTER(vp)]
        L.ffn_b200_st_close.argtypes = [vp]
        L.ffn_b200_st_count.argtypes = [vp]
        L.ffn_b200_st_count.restype = sz
        L.ffn_b200_st_name.argtypes = [vp, sz]
        L.ffn_b200_st_name.restype = C.c_char_p
        L.ffn_b200_st_find.argtypes = [vp, C.c_char_p, C.POINTER(C.c_char_p), C.POINTER(C.c_int64),
                                       C.POINTER(C.c_int), C.POINTER(vp), C.POINTER(sz)]
        L.ffn_b200_st_expert_bytes.argtypes = [vp, C.c_char_p, sz, sz, C.POINTER(C.c_int), C.POINTER(sz)]
        L.ffn_b200_st_load_expert.argtypes = [vp, C.c_char_p, sz, sz, vp, sz, vp, C.POINTER(Expert)]
        _lib = L
    return _lib


def check(rc: int, what: str = "") -> None:
    if rc != 0:
        msg = lib().ffn_b200_last_error().decode(errors="replace")
        raise FfnError(f"{what}: {ERRORS.get(rc, rc)}: {msg}")


def launch_count() -> int:
    return int(lib().ffn_b200_launch_count())


def profile_enable(on: bool) -> None:
    """Start (True: clears the totals) or stop per-kernel event timing."""
    check(lib().ffn_b200_profile_enable(int(on)), "profile_enable")


def profile_kinds(names=None) -> None:
    """Time only these kernel kinds (names from K_NAMES; None: all)."""
    mask = 0xFFFFFFFF if names is None else sum(1 << K_NAMES.index(n) for n in names)
    check(lib().ffn_b200_profile_kinds(C.c_uint32(mask)), "profile_kinds")


def profile_read() -> dict:
    """{kernel kind name: (total device ms, launches)} since profile_enable(True)."""
    out = {}
    for k, name in enumerate(K_NAMES):
        ms, n = C.c_double(), C.c_uint64()
        check(lib().ffn_b200_profile_read(k, C.byref(ms), C.byref(n)), "profile_read")
        if n.value:
            out[name] = (ms.value, int(n.value))
    return out


def key(parent: int, v: int) -> int:
    return int(lib().ffn_b200_key(parent & (2**64 - 1), v))


def path_key(*path: int) -> int:
    """Same key path as the oracle's generator: derive(derive(ROOT, a), b)..."""
    k = 0x464C415348313031
    for v in path:
        k = key(k, int(v))
    return k


# ----------------------------------------------------------- torch glue
def _torch():
    import torch
    return torch


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


class EpExchange:
    """NVLink peer exchange of the expert-parallel partial outputs (one
    process per GPU, torch.distributed initialised).  Every rank's MoE layer
    writes its partial into `part` (residual None); allreduce() then forms
    residual + sum of the parts on every rank."""

    def __init__(self, rank: int, world: int, max_tokens: int, hidden: int, group=None):
        import torch.distributed as dist
        torch = _torch()
        n = int(lib().ffn_b200_ep_handle_bytes())
        h = (C.c_uint8 * n)()
        ep = C.c_void_p()
        check(lib().ffn_b200_ep_create(rank, world, max_tokens, hidden, C.cast(h, C.c_void_p),
                                       C.byref(ep)), "ep_create")
        self.ep = ep
        mine = torch.tensor(list(bytes(h)), dtype=torch.uint8, device="cuda")
        allh = [torch.empty_like(mine) for _ in range(world)]
        dist.all_gather(allh, mine, group=group)
        blob = b"".join(bytes(t.cpu().tolist()) for t in allh)
        buf = (C.c_uint8 * len(blob)).from_buffer_copy(blob)
        check(lib().ffn_b200_ep_connect(ep, C.cast(buf, C.c_void_p)), "ep_connect")
        ptr = int(lib().ffn_b200_ep_part(ep))

        class _View:  # zero-copy torch view of the shared part buffer
            __cuda_array_interface__ = {"shape": (max_tokens, hidden), "typestr": "<f4",
                                        "data": (ptr, False), "version": 2}

        self.part = torch.as_tensor(_View(), device=torch.device("cuda", torch.cuda.current_device()))
        self.hidden = hidden

    def allreduce(self, n_tok: int, residual, out, stream=None):
        check(lib().ffn_b200_ep_allreduce(self.ep, n_tok, _ptr(residual), _ptr(out),
                                          _stream(stream)), "ep_allreduce")
        return out

    def error(self) -> int:
        flag = C.c_int(0)
        check(lib().ffn_b200_ep_error(self.ep, C.byref(flag)), "ep_error")
        return int(flag.value)

    def close(self):
        if self.ep:
            lib().ffn_b200_ep_destroy(self.ep)
            self.ep = None


class Workspace:
    """Grow-only device scratch buffer handed to the library's ws arguments."""

    def __init__(self, device=None):
        self.buf = None
        self.device = device

    def get(self, nbytes: int):
        torch = _torch()
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = None
            self.buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8,
                                   device=self.device or "cuda")
        return self.buf


_ws = {}


def _default_ws(device) -> Workspace:
    d = str(device)
    if d not in _ws:
        _ws[d] = Workspace(device)
    return _ws[d]


# ----------------------------------------------------------- matrices
class Nvfp4Matrix:
    """NVFP4 matrix on the device: w [rows, cols/2] u8, s [rows, cols/16] u8, gs."""

    def __init__(self, w, s, gs: float, rows: int, cols: int):
        self.w, self.s, self.gs, self.rows, self.cols = w, s, float(gs), rows, cols

    def cstruct(self) -> NvMat:
        return NvMat(_ptr(self.w), _ptr(self.s), self.gs, 0)

    @classmethod
    def generate(cls, k: int, rows: int, cols: int, gs: float = 1.0, device="cuda", stream=None):
        torch = _torch()
        w = torch.empty(rows * cols // 2, dtype=torch.uint8, device=device)
        s = torch.empty(rows * cols // 16, dtype=torch.uint8, device=device)
        check(lib().ffn_b200_gen_nvfp4(k, rows, cols, _ptr(w), _ptr(s), _stream(stream)),
              "gen_nvfp4")
        return cls(w, s, gs, rows, cols)

    def matvec(self, x, out=None, stream=None):
        """out [seq, rows] = x [seq, cols] W^T (x float32 CUDA)."""
        torch = _torch()
        x = x.contiguous()
        seq = x.numel() // self.cols
        if out is None:
            out = torch.empty(seq, self.rows, dtype=torch.float32, device=x.device)
        ws = _default_ws(x.device).get(lib().ffn_b200_matvec_ws_bytes(seq, self.cols))
        m = self.cstruct()
        check(lib().ffn_b200_nvfp4_matvec(self.rows, self.cols, seq, C.byref(m), _ptr(x),
                                          _ptr(out), _ptr(ws), ws.numel(), _stream(stream)),
              "nvfp4_matvec")
        return out

    def dequant(self, stream=None):
        torch = _torch()
        out = torch.empty(self.rows, self.cols, dtype=torch.float32, device=self.w.device)
        check(lib().ffn_b200_dequant_nvfp4(self.rows, self.cols, _ptr(self.w), _ptr(self.s),
                                           _ptr(out), _stream(stream)), "dequant_nvfp4")
        return out

    def nbytes(self) -> int:
        return self.w.numel() + self.s.numel()


class Mxfp4Matrix(Nvfp4Matrix):
    """MXFP4 matrix on the device (FMT_MXFP4, flash1017.rs:2674-2747): w
    [rows, cols/2] E2M1 pairs, s [rows, cols/32] E8M0 block scales, gs a power
    of two 2^B taken out of the block scales (1 for the reference's tensors)."""

    @staticmethod
    def bias_for(s_bytes) -> float:
        """gs = 2^B with B = (largest finite block scale byte) - 140: the
        largest block decodes to 2^13 in f16 (E2M1 6 x 2^13 < 65504)."""
        torch = _torch()
        t = s_bytes if torch.is_tensor(s_bytes) else torch.as_tensor(s_bytes)
        t = t[t != 0xFF]
        return 2.0 ** (int(t.max().item()) - 140) if t.numel() else 1.0

    def matvec(self, x, out=None, stream=None):
        torch = _torch()
        x = x.contiguous()
        seq = x.numel() // self.cols
        if out is None:
            out = torch.empty(seq, self.rows, dtype=torch.float32, device=x.device)
        ws = _default_ws(x.device).get(lib().ffn_b200_matvec_ws_bytes(seq, self.cols))
        m = self.cstruct()
        check(lib().ffn_b200_mxfp4_matvec(self.rows, self.cols, seq, C.byref(m), _ptr(x),
                                          _ptr(out), _ptr(ws), ws.numel(), _stream(stream)),
              "mxfp4_matvec")
        return out

    def nbytes(self) -> int:
        return self.w.numel() + self.s.numel()


class Mxfp8Matrix(Nvfp4Matrix):
    """MXFP8 matrix on the device (FMT_MXFP8, the shared expert's format,
    flash1017.rs:1920-1984): w [rows, cols] E4M3, s [ceil(rows/32), cols/32]
    E8M0 scales of 32 x 32 blocks, gs a power of two 2^B taken out of them."""

    @staticmethod
    def bias_for(s_bytes) -> float:
        """gs = 2^B, B = (largest finite scale byte) - 134: the largest block
        decodes to 2^7 in f16 (E4M3 448 x 2^7 < 65504)."""
        torch = _torch()
        t = s_bytes if torch.is_tensor(s_bytes) else torch.as_tensor(s_bytes)
        t = t[t != 0xFF]
        return 2.0 ** (int(t.max().item()) - 134) if t.numel() else 1.0

    def matvec(self, x, out=None, stream=None):
        torch = _torch()
        x = x.contiguous()
        seq = x.numel() // self.cols
        if out is None:
            out = torch.empty(seq, self.rows, dtype=torch.float32, device=x.device)
        ws = _default_ws(x.device).get(lib().ffn_b200_matvec_ws_bytes(seq, self.cols))
        m = self.cstruct()
        check(lib().ffn_b200_mxfp8_matvec(self.rows, self.cols, seq, C.byref(m), _ptr(x),
                                          _ptr(out), _ptr(ws), ws.numel(), _stream(stream)),
              "mxfp8_matvec")
        return out

    def nbytes(self) -> int:
        return self.w.numel() + self.s.numel()


class TernaryMatrix:
    """Packed ternary matrix p [rows, cols/4] u8 + rs [rows] f32 (+ optional
    rank-16 core a [16, cols] i8, a_sc [16], b [rows, 16] i8, b_sc [16]; +
    optional U8 block scales bs [rows, cols/64])."""

    def __init__(self, p, rs, rows, cols, core=None, bs=None):
        self.p, self.rs, self.rows, self.cols, self.core = p, rs, rows, cols, core
        self.bs = bs

    def cstruct(self) -> TnMat:
        c = self.core
        return TnMat(_ptr(self.p), _ptr(self.rs), _ptr(c[0]) if c else None,
                     _ptr(c[1]) if c else None, _ptr(c[2]) if c else None,
                     _ptr(c[3]) if c else None, _ptr(self.bs) if self.bs is not None else None)

    @classmethod
    def generate(cls, k: int, rows: int, cols: int, with_core: bool = True, device="cuda",
                 stream=None):
        torch = _torch()
        p = torch.empty(rows * cols // 4, dtype=torch.uint8, device=device)
        rs = torch.empty(rows, dtype=torch.float32, device=device)
        check(lib().ffn_b200_gen_ternary(k, rows, cols, _ptr(p), _ptr(rs), _stream(stream)),
              "gen_ternary")
        core = None
        if with_core:
            a = torch.empty(16 * cols, dtype=torch.int8, device=device)
            a_sc = torch.empty(16, dtype=torch.float32, device=device)
            b = torch.empty(rows * 16, dtype=torch.int8, device=device)
            b_sc = torch.empty(16, dtype=torch.float32, device=device)
            check(lib().ffn_b200_gen_core(k, rows, cols, _ptr(a), _ptr(a_sc), _ptr(b), _ptr(b_sc),
                                          _stream(stream)), "gen_core")
            core = (a, a_sc, b, b_sc)
        return cls(p, rs, rows, cols, core)

    @classmethod
    def compress(cls, w, s, gs: float, rows: int, cols: int, seed: int, stream=None):
        """The 106 GB format's compressor (ffn_b200_compress_ternary_b64): an
        NVFP4 matrix (device w [rows, cols/2], s [rows, cols/16], per-tensor
        scale gs) -> ternary codes, row scales, U8 block-64 scales and the
        rank-16 Q8 core of the residual."""
        torch = _torch()
        dev = w.device
        p = torch.empty(rows * cols // 4, dtype=torch.uint8, device=dev)
        rs = torch.empty(rows, dtype=torch.float32, device=dev)
        bs = torch.empty(rows * cols // 64, dtype=torch.uint8, device=dev)
        a = torch.empty(16 * cols, dtype=torch.int8, device=dev)
        a_sc = torch.empty(16, dtype=torch.float32, device=dev)
        b = torch.empty(rows * 16, dtype=torch.int8, device=dev)
        b_sc = torch.empty(16, dtype=torch.float32, device=dev)
        ws = _default_ws(dev).get(lib().ffn_b200_compress_ws_bytes(rows, cols))
        check(lib().ffn_b200_compress_ternary_b64(rows, cols, _ptr(w), _ptr(s), float(gs),
                                                  int(seed) & (2**64 - 1), _ptr(p), _ptr(rs),
                                                  _ptr(bs), _ptr(b), _ptr(b_sc), _ptr(a), _ptr(a_sc),
                                                  _ptr(ws), ws.numel(), _stream(stream)),
              "compress_ternary_b64")
        return cls(p, rs, rows, cols, (a, a_sc, b, b_sc), bs)

    def matvec(self, x, out=None, stream=None):
        torch = _torch()
        x = x.contiguous()
        seq = x.numel() // self.cols
        if out is None:
            out = torch.empty(seq, self.rows, dtype=torch.float32, device=x.device)
        ws = _default_ws(x.device).get(lib().ffn_b200_matvec_ws_bytes(seq, self.cols))
        m = self.cstruct()
        check(lib().ffn_b200_ternary_matvec(self.rows, self.cols, seq, C.byref(m), _ptr(x),
                                            _ptr(out), _ptr(ws), ws.numel(), _stream(stream)),
              "ternary_matvec")
        return out

    def dequant(self, stream=None):
        torch = _torch()
        out = torch.empty(self.rows, self.cols, dtype=torch.float32, device=self.p.device)
        check(lib().ffn_b200_dequant_ternary(self.rows, self.cols, _ptr(self.p), _ptr(out),
                                             _stream(stream)), "dequant_ternary")
        return out

    def nbytes(self) -> int:
        n = self.p.numel() + 4 * self.rs.numel()
        if self.bs is not None:
            n += self.bs.numel()
        if self.core:
            n += self.core[0].numel() + self.core[2].numel() + 128
        return n


# Tensor tags of the generator key paths (same values as the oracle's).
TAG_W1, TAG_W3, TAG_W2, TAG_ROUTER, TAG_X, TAG_BIAS = 1, 3, 2, 10, 11, 12


class SwigluExpert:
    """gate (w1), up (w3), down (w2) of one SwiGLU expert on the device."""

    def __init__(self, fmt, mats, inter, hidden, proj_scale=1.0):
        self.fmt, self.mats, self.inter, self.hidden = fmt, mats, inter, hidden
        self.proj_scale = float(proj_scale)
        self.fp4 = None  # (gate/up, down) stage images of the FP4 path

    def cstruct(self) -> Expert:
        e = Expert()
        e.format = self.fmt
        e.proj_scale = self.proj_scale
        for i, m in enumerate(self.mats):
            if self.fmt == FMT_TERNARY:
                e.tn[i] = m.cstruct()
            else:  # NVFP4 and MXFP4 use nv[]
                e.nv[i] = m.cstruct()
        if self.fp4 is not None:
            e.fp4_gu, e.fp4_dn = _ptr(self.fp4[0]), _ptr(self.fp4[1])
        return e

    def pack_fp4(self, gu=None, dn=None, stream=None):
        """The FP4 path's stage images of this NVFP4 expert
        (ffn_b200_pack_nvfp4_expert), into gu / dn (uint8 device tensors of
        ffn_b200_fp4_pack_bytes, e.g. views of one larger buffer) or new
        tensors; raises FfnError when a scale byte is not UE4M3.  Returns self."""
        torch = _torch()
        dev = self.mats[0].w.device
        nb = [lib().ffn_b200_fp4_pack_bytes(self.inter, self.hidden, w) for w in (0, 1)]
        if gu is None:
            gu = torch.empty(nb[0], dtype=torch.uint8, device=dev)
        if dn is None:
            dn = torch.empty(nb[1], dtype=torch.uint8, device=dev)
        if gu.numel() < nb[0] or dn.numel() < nb[1]:
            raise FfnError("pack_fp4: image buffers too small")
        e = self.cstruct()
        check(lib().ffn_b200_pack_nvfp4_expert(self.inter, self.hidden, C.byref(e), _ptr(gu), _ptr(dn),
                                               _stream(stream)), "pack_nvfp4_expert")
        self.fp4 = (gu, dn)
        return self

    @classmethod
    def generate(cls, fmt, seed, layer, expert, inter, hidden, gs=1.0, with_core=True,
                 proj_scale=1.0, device="cuda", stream=None):
        tags = (TAG_W1, TAG_W3, TAG_W2)
        shapes = ((inter, hidden), (inter, hidden), (hidden, inter))
        mats = []
        for tag, (r, c) in zip(tags, shapes):
            k = path_key(seed, layer, expert, tag)
            if fmt == FMT_NVFP4:
                mats.append(Nvfp4Matrix.generate(k, r, c, gs, device, stream))
            else:
                mats.append(TernaryMatrix.generate(k, r, c, with_core, device, stream))
        return cls(fmt, mats, inter, hidden, proj_scale)

    def forward(self, x, out=None, weight=1.0, accumulate=False, stream=None):
        torch = _torch()
        x = x.contiguous()
        seq = x.numel() // self.hidden
        if out is None:
            out = torch.zeros(seq, self.hidden, dtype=torch.float32, device=x.device)
        ws = _default_ws(x.device).get(lib().ffn_b200_expert_ws_bytes(self.inter, self.hidden, seq))
        e = self.cstruct()
        check(lib().ffn_b200_expert_forward(self.inter, self.hidden, seq, C.byref(e), _ptr(x),
                                            _ptr(out), float(weight), int(accumulate), _ptr(ws),
                                            ws.numel(), _stream(stream)), "expert_forward")
        return out

    def nbytes(self) -> int:
        return sum(m.nbytes() for m in self.mats)


class LoadedExpert(SwigluExpert):
    """An expert whose tensors were copied from a shard into one device buffer."""

    def __init__(self, desc: "Expert", buf, inter, hidden):
        super().__init__(desc.format, None, inter, hidden, desc.proj_scale)
        self.desc, self.buf = desc, buf

    def cstruct(self) -> "Expert":
        e = Expert.from_buffer_copy(self.desc)
        e.proj_scale = self.proj_scale
        return e

    def nbytes(self) -> int:
        return int(self.buf.numel())


class SafetensorsShard:
    """A .safetensors shard mapped read-only by the library (ffn_b200_st_*,
    the reference's Flash1017ShardInspector, flash1017.rs:108-235): tensor
    lookup and routed experts copied straight into HBM."""

    def __init__(self, path):
        h = C.c_void_p()
        check(lib().ffn_b200_st_open(os.fsencode(str(path)), C.byref(h)), "st_open")
        self._h = h

    def close(self):
        if self._h:
            lib().ffn_b200_st_close(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def names(self):
        L = lib()
        return [L.ffn_b200_st_name(self._h, i).decode() for i in range(L.ffn_b200_st_count(self._h))]

    def __contains__(self, name) -> bool:
        return name in set(self.names())

    def tensor(self, name):
        """(dtype, shape, bytes): a copy of the tensor's bytes from the mapping."""
        dt, nd, data, nb = C.c_char_p(), C.c_int(), C.c_void_p(), C.c_size_t()
        shape = (C.c_int64 * 8)()
        check(lib().ffn_b200_st_find(self._h, name.encode(), C.byref(dt), shape, C.byref(nd),
                                     C.byref(data), C.byref(nb)), "st_find")
        return dt.value.decode(), tuple(shape[i] for i in range(nd.value)), C.string_at(data, nb.value)

    def expert_bytes(self, prefix, hidden, inter):
        fmt, nb = C.c_int(), C.c_size_t()
        check(lib().ffn_b200_st_expert_bytes(self._h, prefix.encode(), hidden, inter, C.byref(fmt),
                                             C.byref(nb)), "st_expert_bytes")
        return fmt.value, nb.value

    def load_expert(self, prefix, hidden, inter, device="cuda", stream=None) -> LoadedExpert:
        torch = _torch()
        _, nb = self.expert_bytes(prefix, hidden, inter)
        buf = torch.empty(nb + 256, dtype=torch.uint8, device=device)
        off = (-buf.data_ptr()) % 256
        view = buf[off:off + nb]
        e = Expert()
        check(lib().ffn_b200_st_load_expert(self._h, prefix.encode(), hidden, inter, _ptr(view), nb,
                                            _stream(stream), C.byref(e)), "st_load_expert")
        ex = LoadedExpert(e, buf, inter, hidden)
        return ex

    def load_layer(self, layer, n_experts, hidden, inter, device="cuda", stream=None):
        """The routed experts layers.<layer>.ffn.experts.<e> (flash1017.rs:5219-5262)."""
        return [self.load_expert(f"layers.{layer}.ffn.experts.{e}", hidden, inter, device, stream)
                for e in range(n_experts)]


def gen_normal(k: int, n: int, stdev: float = 1.0, device="cuda", stream=None):
    torch = _torch()
    out = torch.empty(n, dtype=torch.float32, device=device)
    check(lib().ffn_b200_gen_normal(k, n, float(stdev), _ptr(out), _stream(stream)),
          "gen_normal")
    return out


def topk(logits, top_k, score_fn=SCORE_SIGMOID, bias=None, stream=None):
    """The MoE layer's top-k step on device logits, [n_tok, n_exp] or partial
    planes [n_part, n_tok, n_exp] (added in plane order): (idx int32, wt f32),
    each [n_tok, top_k] (ffn_b200_topk)."""
    torch = _torch()
    lg = logits if logits.dim() == 3 else logits.unsqueeze(0)
    lg = lg.contiguous()
    n_part, n_tok, n_exp = lg.shape
    idx = torch.empty(n_tok, top_k, dtype=torch.int32, device=lg.device)
    wt = torch.empty(n_tok, top_k, dtype=torch.float32, device=lg.device)
    b = None if bias is None else bias.contiguous()
    check(lib().ffn_b200_topk(n_tok, n_exp, top_k, int(score_fn), _ptr(lg), n_part,
                              None if b is None else _ptr(b), _ptr(idx), _ptr(wt), _stream(stream)),
          "topk")
    return idx, wt


def expert_table(experts, device="cuda"):
    """Device array of ffn_b200_expert structs (None entries: placeholders)."""
    torch = _torch()
    table = (Expert * len(experts))()
    fmts = set()
    for i, e in enumerate(experts):
        if e is not None:
            table[i] = e.cstruct()
            fmts.add(e.fmt)
    return torch.frombuffer(bytearray(bytes(table)), dtype=torch.uint8).to(device), fmts


class MoeLayer:
    """Routed SwiGLU MoE layer over device-resident experts."""

    def __init__(self, experts, router_w, hidden, inter, top_k=6, score_fn=SCORE_SIGMOID,
                 router_bias=None, router_mode=ROUTER_EXACT, expert_range=None, device="cuda",
                 table=None, ws=None, norm_w=None, norm_eps=1e-20, path=PATH_AUTO):
        self.experts = experts  # SwigluExpert list (None allowed outside expert_range)
        self.router_w = router_w
        self.router_bias = router_bias
        self.norm_w = norm_w
        self.hidden, self.inter, self.top_k = hidden, inter, top_k
        n = len(experts)
        if any(e is not None and e.fmt == FMT_MXFP8 for e in experts):
            raise FfnError("MoE tables hold NVFP4, MXFP4 and ternary experts; MXFP8 is for "
                           "dense (shared) experts")
        if table is None:
            self.table, fmts = expert_table(experts, device)
        else:  # a shared (table, formats) pair
            self.table, fmts = table
        # experts kept only as stage images (reference-layout pointers NULL) can
        # run nowhere but the FP4 path
        if any(e is not None and e.mats is not None and any(getattr(m, "w", 0) is None for m in e.mats)
               for e in experts):
            if path not in (PATH_AUTO, PATH_FP4):
                raise FfnError("experts held only as FP4 stage images run only on PATH_FP4")
            path = PATH_FP4
        lo, hi = expert_range if expert_range else (0, n)
        # the FP4 path reads stage images: every local expert must carry them
        # (the table must have been built after pack_fp4)
        packed = all(experts[e] is not None and getattr(experts[e], "fp4", None) is not None
                     for e in range(lo, hi))
        self.desc = MoeDesc(hidden, inter, n, top_k, _ptr(self.table), _ptr(router_w),
                            _ptr(router_bias), score_fn, router_mode, lo, hi,
                            int(FMT_NVFP4 in fmts or FMT_MXFP4 in fmts or not fmts),
                            int(FMT_TERNARY in fmts), _ptr(norm_w), float(norm_eps), int(path),
                            int(FMT_MXFP4 in fmts), int(packed))
        self.ws = ws if ws is not None else Workspace(device)

    def ws_bytes(self, n_tok: int) -> int:
        return int(lib().ffn_b200_moe_ws_bytes(C.byref(self.desc), n_tok))

    def forward_ep(self, exchange, x, out, residual=None, topk_idx=None, topk_w=None, stream=None):
        """This rank's experts (expert_range) with the expert-parallel exchange
        fused in: out = residual + the layer over every rank's experts."""
        x = x.contiguous()
        n_tok = x.numel() // self.hidden
        ws = self.ws.get(self.ws_bytes(n_tok))
        check(lib().ffn_b200_ep_moe_layer(exchange.ep, C.byref(self.desc), n_tok, _ptr(x), _ptr(residual),
                                          _ptr(out), _ptr(topk_idx), _ptr(topk_w), _ptr(ws), ws.numel(),
                                          _stream(stream)), "ep_moe_layer")
        return out

    def forward(self, x, out=None, residual=None, topk_idx=None, topk_w=None, stream=None):
        torch = _torch()
        x = x.contiguous()
        n_tok = x.numel() // self.hidden
        if out is None:
            out = torch.empty(n_tok, self.hidden, dtype=torch.float32, device=x.device)
        ws = self.ws.get(self.ws_bytes(n_tok))
        check(lib().ffn_b200_moe_layer(C.byref(self.desc), n_tok, _ptr(x), _ptr(residual),
                                       _ptr(out), _ptr(topk_idx), _ptr(topk_w), _ptr(ws),
                                       ws.numel(), _stream(stream)), "moe_layer")
        return out


# ------------------------------------------------ activation rows of any type
# The operators below take rows of f32, bf16 or f16: 2-d CUDA tensors whose rows
# may be slices of wider ones.  Rows that are not contiguous inside are copied;
# outputs are written in place.  `stream`: where the kernels run and what is
# returned belongs to (default: the current stream of the tensors' device).
# Temporaries come from torch's allocator, so calls on several streams and
# captured graphs share none.  Nothing here takes part in autograd: the
# gradients are calls of their own.
#
# One call is one or two kernel launches of a few microseconds, so the checks
# stay lean: torch's accessors below cost 0.1 us each, current_stream() 2.
# The plain cases go through a CPython module (csrc/torch_calls.cpp) that makes
# the outputs and calls the library; what it does not take (None) and everything
# where it was not built, or does not load, comes through here.
_dts = None
_T = _dev_now = _raw_stream = _calls = None


def _calls_path():
    """The module built for this Python and this torch."""
    import torch
    return os.path.join(HERE, "_build", f"ffn_b200_torch.{sys.implementation.cache_tag}.torch-{torch.__version__}.so")


def _setup():
    global _T, _dts, _dev_now, _raw_stream, _calls
    import torch
    _dts = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}
    _dev_now, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    lib()
    path = _calls_path()
    if os.path.exists(path):
        import importlib.util
        spec = importlib.util.spec_from_file_location("ffn_b200_torch", path)
        try:
            calls = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(calls)
            _calls = calls
        except ImportError as e:
            import warnings
            warnings.warn(f"{path} does not load, the row operators' calls go through ctypes: {e}", RuntimeWarning,
                          stacklevel=3)
    _T = torch


def _answer(r, what):
    """An entry point's answer through the module: tensors, or its error."""
    if type(r) is int:
        check(r, what)
    return r


def _dtype(dtype):
    d = _dts.get(dtype)
    if d is None:
        raise FfnError(f"rows must be float32, bfloat16 or float16, not {dtype}")
    return d


def _dev(t, stream):
    """t's device index where a call on t can run as it is, -1 where the device
    or the stream has to be switched first."""
    if _T is None:
        _setup()
    d = t.get_device()
    if d < 0:
        raise FfnError("expected CUDA tensors")
    return d if stream is None and d == _dev_now() else -1


def _on(t, stream):
    if stream is None:
        return _T.cuda.device(t.device)
    if stream.device != t.device:
        raise FfnError(f"the stream is on {stream.device}, the tensors on {t.device}")
    return _T.cuda.stream(stream)


def _in(t, what, dev, dtype, rows, cols):
    """(t, row stride) as rows the library reads: 2-d, contiguous inside a row;
    rows or cols None: any."""
    sh = t.shape
    if len(sh) != 2 or (rows is not None and sh[0] != rows) or (cols is not None and sh[1] != cols):
        raise FfnError(f"{what}: expected shape [{'rows' if rows is None else rows}, "
                       f"{'cols' if cols is None else cols}], got {list(sh)}")
    if t.get_device() != dev:
        raise FfnError(f"{what} is on {t.device}, not on cuda:{dev}")
    if t.dtype is not dtype:
        raise FfnError(f"{what}: expected {dtype}, got {t.dtype}")
    ld, one = t.stride()
    if (one != 1 and sh[1] > 1) or (ld < sh[1] and sh[0] > 1):
        return t.contiguous(), sh[1]
    return t, (ld if sh[0] > 1 else max(ld, sh[1]))


def _out(t, what, dev, dtype, rows, cols):
    """(t, row stride) as rows the library writes; t None: new rows."""
    if t is None:
        return _T.empty((rows, cols), dtype=dtype, device=dev), cols
    got, ld = _in(t, what, dev, dtype, rows, cols)
    if got is not t:
        raise FfnError(f"{what}: output rows must be contiguous and must not overlap")
    return t, ld


def _vec(t, what, dev, n, dtype=None):
    """The address of n contiguous values (float32 unless said otherwise)."""
    if t.dtype is not (dtype or _T.float32) or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        raise FfnError(f"{what}: expected {n} contiguous {dtype or _T.float32} values on cuda:{dev}, got "
                       f"{list(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _pos(pos, what, dev):
    """(tokens, top_k, address) of a pos [tokens, top_k]."""
    sh = pos.shape
    if len(sh) != 2 or sh[1] == 0:
        raise FfnError(f"{what}: pos must be int32 [tokens, top_k]")
    return sh[0], sh[1], _vec(pos, "pos", dev, sh[0] * sh[1], _T.int32)


def quantize_int8(x, act=ACT_NONE, codes=None, scales=None, n_rows=None, stream=None):
    """Rows x [rows, cols] (act ACT_SWIGLU: [rows, 2 cols], gate then up) ->
    (codes int8 [rows, cols], scales f32 [rows]), one scale a row
    (ffn_b200_quantize_int8).  New codes are a view of rows padded to 16 bytes,
    as the int8 product takes them.  n_rows: int32 CUDA tensor of one value, the
    rows in use; the rest are left as they were."""
    dev = _dev(x, stream)
    if dev < 0:
        with _on(x, stream):
            return quantize_int8(x, act, codes, scales, n_rows)
    dt = _dtype(x.dtype)
    x, ld = _in(x, "x", dev, x.dtype, None, None)
    rows, cols = x.shape
    if act == ACT_SWIGLU:
        if cols % 2:
            raise FfnError("quantize_int8: ACT_SWIGLU takes an even number of columns")
        cols //= 2
    if codes is None:
        ldc = (cols + 15) // 16 * 16
        codes = _T.empty((rows, ldc), dtype=_T.int8, device=dev)
        if ldc != cols:
            codes = codes[:, :cols]
    else:
        codes, ldc = _out(codes, "codes", dev, _T.int8, rows, cols)
    if scales is None:
        scales = _T.empty((rows,), dtype=_T.float32, device=dev)
    rc = _lib.ffn_b200_quantize_int8(rows, cols, dt, x.data_ptr(), ld, act,
                                     None if n_rows is None else _vec(n_rows, "n_rows", dev, 1, _T.int32),
                                     codes.data_ptr(), ldc, _vec(scales, "scales", dev, rows), _raw_stream(dev))
    if rc:
        check(rc, "quantize_int8")
    return codes, scales


class Int8Matrix:
    """int8 weights on the device, one matrix w [rows, cols] or several experts'
    [groups, rows, cols], with a scale (and optionally a bias) per output
    channel, f32 [(groups,) rows].  The rows of w may be padded (slices of wider
    rows); rows that do not start on 16-byte boundaries are laid out again."""

    def __init__(self, w, scale, bias=None):
        dev = _dev(w, None)
        dev = w.get_device() if dev < 0 else dev
        sh = w.shape
        if w.dtype is not _T.int8 or len(sh) not in (2, 3) or 0 in sh:
            raise FfnError("Int8Matrix: w must be a CUDA int8 tensor [rows, cols] or [groups, rows, cols]")
        st = w.stride()
        if len(sh) == 2:
            sh, st = (1, *sh), (sh[0] * st[0], *st)
            w = w.unsqueeze(0)
        groups, rows, cols = sh
        # the stride between rows, which a single row's tensor need not have
        ld = st[1] if rows > 1 else st[0] if groups > 1 else (cols + 15) // 16 * 16
        if ld % 16 or ld < cols or (cols > 1 and st[2] != 1) or (groups > 1 and st[0] != rows * ld) or w.data_ptr() % 16:
            ld = (cols + 15) // 16 * 16
            wide = _T.zeros((groups, rows, ld), dtype=_T.int8, device=w.device)
            wide[:, :, :cols] = w
            w = wide[:, :, :cols]
        self.groups, self.rows, self.cols, self.w, self.ld, self.device = groups, rows, cols, w, ld, dev
        self.scale, self.bias = scale, bias
        _vec(scale, "scale", dev, groups * rows)
        if bias is not None:
            _vec(bias, "bias", dev, groups * rows)

    @classmethod
    def quantize(cls, w, bias=None, stream=None):
        """Float weights [rows, cols] or [groups, rows, cols], one scale per
        output channel (ffn_b200_quantize_int8 over the channels)."""
        if w.dim() not in (2, 3):
            raise FfnError("Int8Matrix.quantize: w must be [rows, cols] or [groups, rows, cols]")
        if _dev(w, stream) < 0:
            with _on(w, stream):  # reshape copies: on the kernel's stream, in its memory
                return cls.quantize(w, bias)
        codes, scales = quantize_int8(w.reshape(-1, w.shape[-1]))
        ld = (w.shape[-1] + 15) // 16 * 16
        codes = codes.as_strided(w.shape, ((w.shape[1] * ld, ld, 1) if w.dim() == 3 else (ld, 1)))
        return cls(codes, scales, bias)

    def matmul(self, x, out=None, offsets=None, dtype=None, stream=None):
        """out [tokens, rows] = x [tokens, cols] W^T, x float rows (quantised per
        token first) or their (codes, scales); in `dtype`, by default out's
        type, x's, or float32 for codes.  Several groups: offsets int32 [groups
        + 1], tokens offsets[g] .. offsets[g + 1] - 1 take group g, the others'
        rows are left as they were."""
        if _calls is not None and out is None and dtype is None and stream is None and type(x) is not tuple:
            r = _calls.int8_linear(self.w, self.ld, self.scale, self.bias, self.groups, self.rows, self.cols, x,
                                   offsets)
            if r is not None:
                return _answer(r, "int8_matmul")
        floats = not isinstance(x, (tuple, list))
        first = x if floats else x[0]
        dev = _dev(first, stream)
        if dev < 0:
            with _on(first, stream):
                return self.matmul(x, out, offsets, dtype)
        if dev != self.device:
            raise FfnError(f"the weights are on cuda:{self.device}, the tokens on cuda:{dev}")
        k, m, groups = self.cols, self.rows, self.groups
        if dtype is None:
            dtype = out.dtype if out is not None else x.dtype if floats else _T.float32
        x_dtype = x.dtype if floats else _T.int8
        first, ld = _in(first, "x", dev, x_dtype, None, k)
        n = first.shape[0]
        out, ldo = _out(out, "out", dev, dtype, n, m)
        po = None if offsets is None else _vec(offsets, "offsets", dev, groups + 1, _T.int32)
        pb = None if self.bias is None else self.bias.data_ptr()
        if floats:
            nb = _lib.ffn_b200_int8_linear_ws_bytes(n, k, groups, po)
            ws = _T.empty((nb,), dtype=_T.int8, device=dev) if nb else None
            rc = _lib.ffn_b200_int8_linear(n, m, k, groups, po, _dtype(x_dtype), first.data_ptr(), ld,
                                           self.w.data_ptr(), self.ld, self.scale.data_ptr(), pb, _dtype(dtype),
                                           out.data_ptr(), ldo, ws.data_ptr() if nb else None, nb, _raw_stream(dev))
        else:
            if n <= 1:
                ld = (k + 15) // 16 * 16
            if ld % 16 or first.data_ptr() % 16:  # not as quantize_int8 lays them out
                ld = (k + 15) // 16 * 16
                wide = _T.empty((n, ld), dtype=_T.int8, device=dev)
                wide[:, :k] = first
                first = wide
            rc = _lib.ffn_b200_int8_matmul(n, m, k, groups, po, first.data_ptr(), ld, _vec(x[1], "scales", dev, n),
                                           self.w.data_ptr(), self.ld, self.scale.data_ptr(), pb, _dtype(dtype),
                                           out.data_ptr(), ldo, _raw_stream(dev))
        if rc:
            check(rc, "int8_matmul")
        return out

    matvec = matmul

    def dequant(self):
        """f32 weights [(groups,) rows, cols]."""
        w = self.w.float() * self.scale.view(self.groups, self.rows, 1)
        return w[0] if self.groups == 1 else w

    def nbytes(self) -> int:
        return self.groups * self.rows * (self.cols + 4 + (0 if self.bias is None else 4))


def moe_sort(idx, expert_begin, expert_end, stream=None):
    """The routed pairs of idx int32 [tokens, top_k] sorted by expert, those of
    the experts [expert_begin, expert_end) only: (offsets [experts + 1], pos
    [tokens, top_k] with -1 elsewhere, src [tokens * top_k] with -1 behind the
    last row), all int32 (ffn_b200_moe_sort)."""
    if _calls is not None and stream is None:
        r = _calls.moe_sort(idx, expert_begin, expert_end)
        if r is not None:
            return _answer(r, "moe_sort")
    dev = _dev(idx, stream)
    if dev < 0:
        with _on(idx, stream):
            return moe_sort(idx, expert_begin, expert_end)
    sh = idx.shape
    if len(sh) != 2 or idx.dtype is not _T.int32 or sh[1] == 0:
        raise FfnError("moe_sort: idx must be int32 [tokens, top_k]")
    if expert_end <= expert_begin:
        raise FfnError("moe_sort: empty expert range")
    if not idx.is_contiguous():
        idx = idx.contiguous()
    offsets = _T.empty((expert_end - expert_begin + 1,), dtype=_T.int32, device=dev)
    pos = _T.empty_like(idx)
    src = _T.empty((sh[0] * sh[1],), dtype=_T.int32, device=dev)
    rc = _lib.ffn_b200_moe_sort(sh[0], sh[1], idx.data_ptr(), expert_begin, expert_end, offsets.data_ptr(),
                                pos.data_ptr(), src.data_ptr(), _raw_stream(dev))
    if rc:
        check(rc, "moe_sort")
    return offsets, pos, src


def moe_permute(x, pos, out=None, scales=None, out_scales=None, stream=None):
    """out[pos[t, k]] = x[t] for rows of any type (ffn_b200_moe_permute); new
    rows: one per pair.  With scales f32 [tokens] (int8 rows): (out,
    out_scales).  Rows that no pair names are left as they were."""
    if _calls is not None and stream is None and scales is None and out_scales is None:
        r = _calls.moe_permute(x, pos, out)
        if r is not None:
            return _answer(r, "moe_permute")
    dev = _dev(x, stream)
    if dev < 0:
        with _on(x, stream):
            return moe_permute(x, pos, out, scales, out_scales)
    n, top_k, pp = _pos(pos, "moe_permute", dev)
    x, ld = _in(x, "x", dev, x.dtype, n, None)
    cols, es = x.shape[1], x.element_size()
    if out is None:
        # int8 codes as quantize_int8 lays them out keep their padded rows
        ldo = (cols + 15) // 16 * 16 if x.dtype is _T.int8 and ld % 16 == 0 else cols
        out = _T.empty((n * top_k, ldo), dtype=x.dtype, device=dev)
        if ldo != cols:
            out = out[:, :cols]
        rows = n * top_k
    else:
        rows = out.shape[0]
        out, ldo = _out(out, "out", dev, x.dtype, rows, cols)
    ps = pos_out = None
    if scales is not None:
        ps = _vec(scales, "scales", dev, n)
        if out_scales is None:
            out_scales = _T.empty((rows,), dtype=_T.float32, device=dev)
        pos_out = _vec(out_scales, "out_scales", dev, rows)
    elif out_scales is not None:
        raise FfnError("moe_permute: out_scales without scales")
    rc = _lib.ffn_b200_moe_permute(n, top_k, cols * es, x.data_ptr(), ld * es, pp, rows, out.data_ptr(), ldo * es,
                                   ps, pos_out, _raw_stream(dev))
    if rc:
        check(rc, "moe_permute")
    return out if scales is None else (out, out_scales)


def moe_combine(y, pos, weight=None, residual=None, out=None, stream=None):
    """out[t] = residual[t] + sum_k weight[t, k] y[pos[t, k]] (weight f32
    [tokens, top_k] or None: 1), in f32, rounded once (ffn_b200_moe_combine)."""
    if _calls is not None and stream is None and out is None:
        r = _calls.moe_combine(y, pos, weight, residual)
        if r is not None:
            return _answer(r, "moe_combine")
    dev = _dev(y, stream)
    if dev < 0:
        with _on(y, stream):
            return moe_combine(y, pos, weight, residual, out)
    dtype = y.dtype
    dt = _dtype(dtype)
    n, top_k, pp = _pos(pos, "moe_combine", dev)
    y, ld = _in(y, "y", dev, dtype, None, None)
    rows, cols = y.shape
    pr, ldr = None, 0
    if residual is not None:
        residual, ldr = _in(residual, "residual", dev, dtype, n, cols)
        pr = residual.data_ptr()
    out, ldo = _out(out, "out", dev, dtype, n, cols)
    rc = _lib.ffn_b200_moe_combine(n, top_k, cols, dt, y.data_ptr(), ld, rows, pp,
                                   None if weight is None else _vec(weight, "weight", dev, n * top_k), pr, ldr,
                                   out.data_ptr(), ldo, _raw_stream(dev))
    if rc:
        check(rc, "moe_combine")
    return out


def moe_combine_backward(dout, y, pos, weight=None, dy=None, stream=None):
    """Gradients of moe_combine: (dy, dw), dy[pos[t, k]] = weight[t, k] dout[t],
    dw [tokens, top_k] f32 (ffn_b200_moe_combine_bwd).  The residual's gradient
    is dout.  A new dy has zeros in the rows that no pair names; in a given one
    they are left as they were.  No two pairs may name the same row (moe_sort's
    never do)."""
    dev = _dev(y, stream)
    if dev < 0:
        with _on(y, stream):
            return moe_combine_backward(dout, y, pos, weight, dy)
    dtype = y.dtype
    dt = _dtype(dtype)
    n, top_k, pp = _pos(pos, "moe_combine_backward", dev)
    y, ld = _in(y, "y", dev, dtype, None, None)
    rows, cols = y.shape
    dout, ldd = _in(dout, "dout", dev, dtype, n, cols)
    if dy is None:
        dy = _T.zeros((rows, cols), dtype=dtype, device=dev)
    dy, ldy = _out(dy, "dy", dev, dtype, rows, cols)
    dw = _T.empty((n, top_k), dtype=_T.float32, device=dev)
    rc = _lib.ffn_b200_moe_combine_bwd(n, top_k, cols, dt, dout.data_ptr(), ldd, y.data_ptr(), ld, rows, pp,
                                       None if weight is None else _vec(weight, "weight", dev, n * top_k),
                                       dy.data_ptr(), ldy, dw.data_ptr(), _raw_stream(dev))
    if rc:
        check(rc, "moe_combine_bwd")
    return dy, dw


def moe_permute_backward(dout, pos, dx=None, stream=None):
    """Gradient of moe_permute: dx[t] = sum_k dout[pos[t, k]]."""
    return moe_combine(dout, pos, out=dx, stream=stream)


class BlockNorm:
    """The norms after one block and before the next (ffn_b200_block_norm):
    h = alpha residual + beta gate rms(y) post_w, xn = rms(h) pre_w.  post_w
    None: y itself; pre_w None: no xn.  The gate is f32 [cols] (a parameter) or
    [rows, 1] (one per token)."""

    def __init__(self, pre_w=None, post_w=None, alpha=1.0, beta=1.0, eps=1e-6):
        self.pre_w, self.post_w = pre_w, post_w
        self.alpha, self.beta, self.eps = alpha, beta, eps

    def _desc(self, dev, dtype, rows, cols, gate, post):
        kind, pg, pp, pq = GATE_NONE, None, None, None
        if gate is not None:
            sh = gate.shape
            if len(sh) == 1 and sh[0] == cols:
                kind = GATE_CHANNEL
            elif len(sh) == 2 and sh[0] == rows and sh[1] == 1:
                kind = GATE_TOKEN
            else:
                raise FfnError(f"gate: expected [{cols}] or [{rows}, 1], got {list(sh)}")
            pg = _vec(gate, "gate", dev, gate.numel())
        if post and self.post_w is not None:
            pp = _vec(self.post_w, "post_w", dev, cols)
        if self.pre_w is not None:
            pq = _vec(self.pre_w, "pre_w", dev, cols)
        return BlockNormDesc(rows, cols, _dtype(dtype), kind, pp, pg, pq, self.alpha, self.beta, self.eps, 0)

    def forward(self, y, residual=None, gate=None, h=None, xn=None, codes=False, stream=None):
        """(h, xn), each a new tensor or the one given; y None: the residual
        alone.  codes True: (h, xn, codes, scales) with xn None unless given and
        the int8 codes of xn (quantize_int8 of its f32 values)."""
        if _calls is not None and y is not None and h is None and xn is None and not codes and stream is None:
            r = _calls.block_norm(self.pre_w, self.post_w, self.alpha, self.beta, self.eps, y, residual, gate)
            if r is not None:
                return _answer(r, "block_norm")
        like = residual if y is None else y
        if like is None:
            raise FfnError("BlockNorm: neither y nor residual")
        dev = _dev(like, stream)
        if dev < 0:
            with _on(like, stream):
                return self.forward(y, residual, gate, h, xn, codes)
        sh, dtype = like.shape, like.dtype
        if len(sh) != 2:
            raise FfnError(f"BlockNorm: expected rows [rows, cols], got {list(sh)}")
        rows, cols = sh
        if y is None and gate is not None:
            raise FfnError("BlockNorm: a gate without y")
        d = self._desc(dev, dtype, rows, cols, gate, y is not None)
        py, ldy, pr, ldr, px, ldx, pq, ldq, ps = None, 0, None, 0, None, 0, None, 0, None
        if y is not None:
            y, ldy = _in(y, "y", dev, dtype, rows, cols)
            py = y.data_ptr()
        if residual is not None:
            residual, ldr = _in(residual, "residual", dev, dtype, rows, cols)
            pr = residual.data_ptr()
        h, ldh = _out(h, "h", dev, dtype, rows, cols)
        if xn is not None or (self.pre_w is not None and not codes):
            xn, ldx = _out(xn, "xn", dev, dtype, rows, cols)
            px = xn.data_ptr()
        q = sc = None
        if codes:
            if self.pre_w is None:
                raise FfnError("BlockNorm: codes need pre_w")
            ldq = (cols + 15) // 16 * 16
            q = _T.empty((rows, ldq), dtype=_T.int8, device=dev)[:, :cols]
            sc = _T.empty((rows,), dtype=_T.float32, device=dev)
            pq, ps = q.data_ptr(), sc.data_ptr()
        rc = _lib.ffn_b200_block_norm(C.byref(d), py, ldy, pr, ldr, h.data_ptr(), ldh, px, ldx, pq, ldq, ps,
                                      _raw_stream(dev))
        if rc:
            check(rc, "block_norm")
        return (h, xn, q, sc) if codes else (h, xn)

    def backward(self, y, h, dh=None, dxn=None, gate=None, stream=None):
        """The gradients, from the y and h of the forward pass and the gradients
        of h (past the norm) and xn: {"dy", "dres", "dpost_w", "dgate",
        "dpre_w"}, None where there is no such input."""
        like = dh if dxn is None else dxn
        if like is None:
            raise FfnError("BlockNorm.backward: neither dh nor dxn")
        dev = _dev(like, stream)
        if dev < 0:
            with _on(like, stream):
                return self.backward(y, h, dh, dxn, gate)
        sh, dtype = like.shape, like.dtype
        if len(sh) != 2:
            raise FfnError(f"BlockNorm.backward: expected rows [rows, cols], got {list(sh)}")
        rows, cols = sh
        if y is None and gate is not None:
            raise FfnError("BlockNorm.backward: a gate without y")
        if dxn is not None and (h is None or self.pre_w is None):
            raise FfnError("BlockNorm.backward: dxn needs h and pre_w")
        d = self._desc(dev, dtype, rows, cols, gate, y is not None)
        keep, at = [], []  # rows that were copied live until the call
        for t, what in ((y, "y"), (h, "h"), (dh, "dh"), (dxn, "dxn")):
            if t is None:
                at += [None, 0]
            else:
                t, ld = _in(t, what, dev, dtype, rows, cols)
                keep.append(t)
                at += [t.data_ptr(), ld]

        def new(on, shape, dtype):
            return _T.empty(shape, dtype=dtype, device=dev) if on else None
        f32 = _T.float32
        dres = new(True, (rows, cols), dtype)
        dy = new(y is not None, (rows, cols), dtype)
        dpost = new(d.post_w is not None, (cols,), f32)
        dgate = None if gate is None else _T.empty_like(gate)
        dpre = new(dxn is not None, (cols,), f32)
        nb = _lib.ffn_b200_block_norm_bwd_ws_bytes(C.byref(d))
        ws = new(True, (nb,), _T.uint8)
        rc = _lib.ffn_b200_block_norm_bwd(C.byref(d), *at, dres.data_ptr(), cols, _ptr(dy), cols, _ptr(dpost),
                                          _ptr(dgate), _ptr(dpre), ws.data_ptr(), nb, _raw_stream(dev))
        if rc:
            check(rc, "block_norm_bwd")
        return {"dy": dy, "dres": dres, "dpost_w": dpost, "dgate": dgate, "dpre_w": dpre}


class Int8Experts:
    """SwiGLU experts in int8 behind a router: gate_up Int8Matrix [experts,
    2 inter, hidden] (gate channels, then up), down Int8Matrix [experts, hidden,
    inter], those of the experts [expert_begin, expert_begin + experts) of the
    routing (expert parallelism: the others' contributions are left out)."""

    def __init__(self, gate_up, down, expert_begin=0):
        if gate_up.groups != down.groups or gate_up.rows != 2 * down.cols or gate_up.cols != down.rows:
            raise FfnError("Int8Experts: expected gate_up [experts, 2 inter, hidden] and down "
                           "[experts, hidden, inter]")
        self.gate_up, self.down, self.expert_begin = gate_up, down, int(expert_begin)

    def forward(self, x, topk_idx, topk_w, residual=None, out=None, stream=None):
        """out[t] = residual[t] + sum_k topk_w[t, k] expert(topk_idx[t, k])(x[t]);
        x float rows [tokens, hidden], or the (codes, scales) of such rows with
        `residual` or `out` giving the type (float32 without either)."""
        first = x[0] if isinstance(x, (tuple, list)) else x
        if _dev(first, stream) < 0:
            with _on(first, stream):
                return self.forward(x, topk_idx, topk_w, residual, out)
        like = next((t for t in (x if first is x else None, residual, out) if t is not None), None)
        dtype = _T.float32 if like is None else like.dtype
        codes, scales = quantize_int8(x) if first is x else x
        offsets, pos, _ = moe_sort(topk_idx, self.expert_begin, self.expert_begin + self.gate_up.groups)
        rows = moe_permute(codes, pos, scales=scales)
        gu = self.gate_up.matmul(rows, offsets=offsets, dtype=dtype)
        act = quantize_int8(gu, ACT_SWIGLU, n_rows=offsets[-1:])
        y = self.down.matmul(act, offsets=offsets, dtype=dtype)
        return moe_combine(y, pos, topk_w, residual=residual, out=out)
