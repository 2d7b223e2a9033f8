"""Python binding of the B200-native MiniMax-M2.7 MoE hot path (ctypes over the C ABI).

The compute lives in lib/libminimax_moe.so (hand-written sm_100a CUDA, see csrc/).  This module
only declares the C prototypes of include/minimax_moe.h and offers thin helpers that take torch
CUDA tensors.  There is no CPU fallback: every entry point raises when the library is missing.

The directory name contains a dash, so import it by path:

    import importlib.util, sys
    spec = importlib.util.spec_from_file_location("minimax_rs_b200", "<repo>/minimax-rs_b200/__init__.py",
                                                  submodule_search_locations=["<repo>/minimax-rs_b200"])
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
LIB_PATH = PKG_DIR / "lib" / "libminimax_moe.so"
HEADER = PKG_DIR.parent / "include" / "minimax_moe.h"

MMRS_OK, MMRS_ERR_ARG, MMRS_ERR_UNSUPPORTED, MMRS_ERR_LAUNCH, MMRS_ERR_TIMEOUT, MMRS_ERR_ALLOC = range(6)
MMRS_ERR_SCRATCH_LIMIT = 6
MMRS_ERR_NONFINITE = 7
Q8_0, Q4K, Q2K, Q3K, Q5K, Q6K = 0, 1, 2, 3, 4, 5
ERROR_NAMES = {0: "ok", 1: "invalid argument", 2: "unsupported", 3: "launch failure", 4: "device wait timed out",
               5: "allocation failure", 6: "problem exceeds the fixed scratch", 7: "non-finite value"}


class MoeError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: {ERROR_NAMES.get(code, code)} ({code})")
        self.code = code


class MmrsMoeWeights(C.Structure):
    _fields_ = [("router", C.c_void_p), ("bias", C.c_void_p), ("gate", C.c_void_p), ("up", C.c_void_p),
                ("down", C.c_void_p), ("gate_up_type", C.c_int), ("down_type", C.c_int),
                ("num_experts", C.c_int), ("topk", C.c_int), ("hidden", C.c_int), ("inter", C.c_int)]


class MmrsPeerGroup(C.Structure):
    _fields_ = [("world", C.c_int), ("rank", C.c_int), ("mine", C.c_void_p), ("peers", C.c_void_p * 8),
                ("ar_capacity", C.c_size_t), ("expert_parallel", C.c_int)]


_VP, _I, _U32, _U64, _I64, _F = C.c_void_p, C.c_int, C.c_uint32, C.c_uint64, C.c_int64, C.c_float
_SZ = C.c_size_t


class MmrsLmHead(C.Structure):
    _fields_ = [("weight", C.c_void_p), ("norm_weight", C.c_void_p), ("vocab", C.c_int), ("hidden", C.c_int),
                ("eps", C.c_float)]


class MmrsSamplingParams(C.Structure):
    """include/minimax_sample.h: SamplingParams (src/sampling.rs:13-17)."""
    _fields_ = [("temperature", C.c_double), ("top_p", C.c_double), ("top_k", C.c_int)]


class MmrsAttnWeights(C.Structure):
    """include/minimax_attn.h: MmrsAttnWeights."""
    _fields_ = [("wq", C.c_void_p), ("wk", C.c_void_p), ("wv", C.c_void_p), ("wo", C.c_void_p),
                ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("rope_cos", C.c_void_p), ("rope_sin", C.c_void_p),
                ("hidden", C.c_int), ("query_heads", C.c_int), ("kv_heads", C.c_int), ("rope_dim", C.c_int),
                ("max_positions", C.c_int), ("eps", C.c_float)]


class MmrsPagedCache(C.Structure):
    """include/minimax_paged.h: MmrsPagedCache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("num_pages", C.c_int), ("page_size", C.c_int), ("kv_heads", C.c_int)]


class MmrsPagedBatch(C.Structure):
    """include/minimax_paged.h: MmrsPagedBatch."""
    _fields_ = [("cu_q", C.c_void_p), ("seq_len", C.c_void_p), ("page_table", C.c_void_p), ("num_seqs", C.c_int),
                ("table_stride", C.c_int), ("total_q", C.c_int), ("max_q", C.c_int), ("max_len", C.c_int)]


# name -> (restype, argtypes)
PROTOTYPES = {
    "minimax_moe_decode_topk": (None, [_VP] * 7),
    "moe_gemm_gguf_decode_silu": (None, [_VP] * 8 + [_I] * 6 + [_VP]),
    "moe_gemm_gguf": (None, [_VP] * 6 + [_I] * 6 + [_VP]),
    "moe_gemm_mmq_gguf": (None, [_VP] * 6 + [_I] * 6 + [_VP]),
    "moe_sort_routes": (None, [_VP] * 3 + [_I] * 2 + [_VP]),
    "mmrs_last_error": (_I, []),
    # decode attention (include/minimax_attn.h)
    "launch_mmvq_gguf_quantize_q8_1_f32": (None, [_VP, _VP, _I, _I, _I, _VP]),
    "launch_mmvq_gguf_q8_0_f32_plain": (None, [_VP] * 3 + [_I] * 5 + [_VP]),
    "launch_mmvq_gguf_qkv_q8_0_f32": (None, [_VP] * 6 + [_I] * 5 + [_VP]),
    "launch_mmvq_gguf_qkv_q8_0_f32_rmsnorm_f16": (None, [_VP] * 9 + [_I] * 5 + [_F, _VP]),
    "launch_partial_rope_f16": (None, [_VP] * 5 + [_I] * 5 + [_VP]),
    "launch_qkv_tp_sumsq_f32": (None, [_VP] * 3 + [_I] * 2 + [_VP]),
    "launch_qkv_tp_rmsnorm_rope_f16": (None, [_VP] * 9 + [_I] * 8 + [_F, _VP]),
    "launch_gqa_decode_mma_f16_128": (None, [_VP] * 5 + [_I] * 7 + [_F, _I, _VP]),
    "mmrs_attn_workspace_bytes": (_SZ, [C.POINTER(MmrsAttnWeights)]),
    "mmrs_attn_workspace_status": (_I, [_VP]),
    "launch_mmvq_gguf_q6_k_f32_plain": (None, [_VP] * 3 + [_I] * 5 + [_VP]),
    "mmrs_lm_head_workspace_bytes": (_SZ, [C.POINTER(MmrsLmHead)]),
    "mmrs_lm_head_workspace_status": (_I, [_VP]),
    "mmrs_lm_head_forward": (_I, [C.POINTER(MmrsLmHead), _VP, _VP, _VP, _VP, _SZ, _VP]),
    "mmrs_rmsnorm_f32": (_I, [_VP, _VP, _VP, _I, _I, _F, _VP]),
    # token sampling (include/minimax_sample.h)
    "mmrs_sample_workspace_bytes": (_SZ, [_I]),
    "mmrs_sample_workspace_status": (_I, [_VP]),
    "mmrs_sample_token": (_I, [_VP, _I, C.POINTER(MmrsSamplingParams), C.c_double, _VP, _VP, _SZ, _VP]),
    "mmrs_token_logprob": (_I, [_VP, _I, _I, _VP, _VP, _SZ, _VP]),
    "mmrs_verify_workspace_bytes": (_SZ, [_I, _I]),
    "mmrs_verify_workspace_status": (_I, [_VP]),
    "mmrs_verify_drafts": (_I, [_VP, _I, _I, _VP, _I, _I, _I] + [_VP] * 9 + [_SZ, _VP]),
    "mmrs_verify_drafts_n": (_I, [_VP, _I, _I, _VP, _I, _I, _I] + [_VP] * 3 + [_I] + [_VP] * 6 + [_SZ, _VP]),
    # paged 8-bit cache (include/minimax_paged.h)
    "mmrs_paged_append": (_I, [C.POINTER(MmrsPagedCache), C.POINTER(MmrsPagedBatch), _VP, _VP, _VP, _I64, _I64, _I64,
                               _I, _I, _VP, _VP, _I, _I, _VP, _I, _VP]),
    "mmrs_paged_attend_workspace_bytes": (_SZ, [_I] * 4),
    "mmrs_paged_attend_status": (_I, [_VP]),
    "mmrs_paged_attend": (_I, [C.POINTER(MmrsPagedCache), C.POINTER(MmrsPagedBatch), _VP, _I64, _I, _I, _F, _I, _I,
                               _VP, _VP, _VP, _SZ, _VP]),
    "mmrs_attn_decode_forward": (_I, [C.POINTER(MmrsAttnWeights), _VP, _VP, _I, _VP, _VP, _VP, _VP, _SZ, _VP]),
    "launch_tp2_peer_all_reduce_f32": (None, [_VP] * 8 + [C.c_uint, _I, _F, _VP]),
    "launch_tp2_peer_broadcast_f32": (None, [_VP] * 4 + [C.c_uint, _I, _I, _VP]),
    "mmrs_xch_bytes": (_SZ, [_SZ]),
    "mmrs_peer_alloc": (_I, [_SZ, C.POINTER(C.c_void_p)]),
    "mmrs_peer_free": (_I, [_VP]),
    "mmrs_ipc_handle": (_I, [_VP, C.POINTER(C.c_uint8)]),
    "mmrs_ipc_open": (_I, [C.POINTER(C.c_uint8), C.POINTER(C.c_void_p)]),
    "mmrs_ipc_close": (_I, [_VP]),
    "mmrs_peer_enable": (_I, [_I]),
    "mmrs_xch_ar_buffer": (_VP, [C.POINTER(MmrsPeerGroup), _U32]),
    "mmrs_peer_all_reduce": (_I, [C.POINTER(MmrsPeerGroup), _VP, _VP, _SZ, _U32, _VP]),
    "mmrs_peer_status": (_I, [C.POINTER(MmrsPeerGroup), _VP]),
    "mmrs_moe_block_forward_group": (_I, [C.POINTER(MmrsMoeWeights), C.POINTER(MmrsPeerGroup), _VP, _VP, _VP, _I,
                                          _VP, _VP, _VP, _SZ, _U32, _VP]),
    "mmrs_moe_block_forward_group_host": (_I, [C.POINTER(MmrsMoeWeights), C.POINTER(MmrsPeerGroup), _VP, _VP, _VP,
                                               _I, _VP, _VP, _VP, _VP, _VP, _SZ, _U32, _VP]),
    "mmrs_moe_workspace_bytes": (_SZ, [C.POINTER(MmrsMoeWeights), _I]),
    "mmrs_moe_workspace_zero_bytes": (_SZ, [C.POINTER(MmrsMoeWeights)]),
    "mmrs_int8_tensor_peak": (_I, [_I, _I, C.POINTER(C.c_double), _VP]),
    "mmrs_moe_block_forward": (_I, [C.POINTER(MmrsMoeWeights), _VP, _VP, _VP, _I, _VP, _VP, _VP, _SZ, _VP]),
    "mmrs_moe_block_forward_host": (_I, [C.POINTER(MmrsMoeWeights), _VP, _VP, _VP, _I, _VP, _VP, _VP, _VP, _VP, _SZ,
                                         _VP]),
    "mmrs_moe_workspace_status": (_I, [_VP, _VP]),
    "mmrs_moe_block_decode_static": (_I, [C.POINTER(MmrsMoeWeights), _VP, _VP, _VP, _VP, _VP, _VP]),
    "mmrs_moe_static_status": (_I, [_VP]),
    "mmrs_moe_workspace_trace": (_I, [_VP, _VP, _I, _VP]),
    "mmrs_synth_normal_f32": (_I, [_VP, _I64, _U64, _U32, _F, _I, _VP]),
    "mmrs_synth_kquant": (_I, [_VP, _I, _U64, _U32] + [_I] * 7 + [_VP]),
}

_lib = None


def lib() -> C.CDLL:
    """Loads the CUDA library (raises if it has not been built: there is no fallback)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: run `python minimax-rs_b200/build.py` "
                               "(the MoE path has no CPU fallback)")
        l = C.CDLL(str(LIB_PATH))
        for name, (res, args) in PROTOTYPES.items():
            f = getattr(l, name)
            f.restype = res
            f.argtypes = args
        _lib = l
    return _lib


def check(code: int, what: str) -> None:
    if code != MMRS_OK:
        raise MoeError(code, what)


def last_error() -> int:
    return lib().mmrs_last_error()


# ---------------------------------------------------------------------------------------------
# torch helpers
# ---------------------------------------------------------------------------------------------
def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> int:
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def row_bytes(gguf_type: int, k: int) -> int:
    return (k // 256) * (176 if gguf_type == Q5K else 144)


class MoeLayer:
    """Device-resident weights of one MoE layer + the C struct that points at them."""

    def __init__(self, router, bias, gate, up, down, gate_up_type: int, down_type: int, topk: int = 8):
        self.router, self.bias, self.gate, self.up, self.down = router, bias, gate, up, down
        self.num_experts, self.hidden = router.shape
        self.inter = gate.numel() // (self.num_experts * row_bytes(gate_up_type, self.hidden))
        self.c = MmrsMoeWeights(router.data_ptr(), bias.data_ptr(), gate.data_ptr(), up.data_ptr(),
                                down.data_ptr(), gate_up_type, down_type, self.num_experts, topk,
                                self.hidden, self.inter)
        self.topk = topk
        self._ws = None

    def workspace(self, max_tokens: int):
        import torch
        nbytes = lib().mmrs_moe_workspace_bytes(C.byref(self.c), max_tokens)
        if self._ws is None or self._ws.numel() < nbytes:
            self._ws = torch.zeros(nbytes, dtype=torch.uint8, device=self.router.device)
        return self._ws

    def forward(self, x, residual=None, y=None, topk_ids=None, topk_w=None, stream=None):
        """y = MoE(x) (+ residual); x [T, hidden] f32 CUDA tensor."""
        import torch
        T = x.shape[0]
        if y is None:
            y = torch.empty_like(x)
        ws = self.workspace(T)
        rc = lib().mmrs_moe_block_forward(C.byref(self.c), x.data_ptr(), _ptr(residual), y.data_ptr(), T,
                                          _ptr(topk_ids), _ptr(topk_w), ws.data_ptr(), ws.numel(), _stream(stream))
        check(rc, "mmrs_moe_block_forward")
        return y

    def forward_host(self, x_host, y_host, x_dev, y_dev, residual=None, topk_ids=None, topk_w=None, stream=None):
        """y_host = MoE(x_host) (+ residual) in one library call: the copy of x_host [T, hidden]
        (pinned host memory) into x_dev, the block into y_dev and the copy back into y_host are
        enqueued on `stream`; residual / topk_* are CUDA tensors as in forward()."""
        T = x_host.shape[0]
        ws = self.workspace(T)
        rc = lib().mmrs_moe_block_forward_host(C.byref(self.c), x_host.data_ptr(), _ptr(residual), y_host.data_ptr(),
                                               T, x_dev.data_ptr(), y_dev.data_ptr(), _ptr(topk_ids), _ptr(topk_w),
                                               ws.data_ptr(), ws.numel(), _stream(stream))
        check(rc, "mmrs_moe_block_forward_host")
        return y_host

    def trace(self, stream=None):
        """Per-CTA phase timestamps (ns) of the last single-token launch: array [256, 32]."""
        import numpy as np
        out = np.zeros(256 * 32, dtype=np.uint64)
        n = lib().mmrs_moe_workspace_trace(self._ws.data_ptr(), out.ctypes.data, out.size, _stream(stream))
        if n < 0:
            raise MoeError(-n, "mmrs_moe_workspace_trace")
        return out.reshape(256, 32)

    def status(self, stream=None) -> int:
        return lib().mmrs_moe_workspace_status(self._ws.data_ptr(), _stream(stream)) if self._ws is not None else 0


def moe_gemm(inp, weights, sorted_token_ids, expert_ids, topk_weights, out, num_experts: int, topk: int,
             size_n: int, size_k: int, gguf_type: int, mmq: bool = False, stream=None):
    """moe_gemm_gguf / moe_gemm_mmq_gguf through the reference ABI; raises on a recorded error."""
    fn = lib().moe_gemm_mmq_gguf if mmq else lib().moe_gemm_gguf
    fn(inp.data_ptr(), weights.data_ptr(), sorted_token_ids.data_ptr(), expert_ids.data_ptr(), _ptr(topk_weights),
       out.data_ptr(), num_experts, topk, sorted_token_ids.numel(), size_n, size_k, gguf_type, _stream(stream))
    check(last_error(), "moe_gemm_mmq_gguf" if mmq else "moe_gemm_gguf")
    return out


def sort_routes(expert_ids, end_bit: int, stream=None):
    """moe_sort_routes: stable sort of u32 keys on bits [0, end_bit) -> (sorted keys, positions)."""
    import torch
    n = expert_ids.numel()
    keys = torch.empty(n, dtype=torch.int32, device=expert_ids.device)
    routes = torch.empty(n, dtype=torch.int32, device=expert_ids.device)
    lib().moe_sort_routes(expert_ids.data_ptr(), keys.data_ptr(), routes.data_ptr(), n, end_bit, _stream(stream))
    check(last_error(), "moe_sort_routes")
    return keys, routes


def int8_tensor_peak(chunks: int = 4096, reps: int = 5, stream=None) -> float:
    """Measured dense int8 tensor-core throughput of the current device, TOPS (mmrs_int8_tensor_peak)."""
    out = C.c_double(0.0)
    check(lib().mmrs_int8_tensor_peak(chunks, reps, C.byref(out), _stream(stream)), "mmrs_int8_tensor_peak")
    return out.value


def synth_normal(t, seed: int, stream_id: int, scale: float = 1.0, bf16: bool = False, stream=None):
    check(lib().mmrs_synth_normal_f32(t.data_ptr(), t.numel(), seed, stream_id, scale, int(bf16), _stream(stream)),
          "mmrs_synth_normal_f32")
    return t


def synth_kquant(t, gguf_type: int, seed: int, stream_id: int, experts: int, rows: int, k: int,
                 row0: int = 0, nrows: int | None = None, kblk0: int = 0, nkblk: int | None = None, stream=None):
    nrows = rows - row0 if nrows is None else nrows
    nkblk = k // 256 - kblk0 if nkblk is None else nkblk
    check(lib().mmrs_synth_kquant(t.data_ptr(), gguf_type, seed, stream_id, experts, rows, k, row0, nrows, kblk0,
                                  nkblk, _stream(stream)), "mmrs_synth_kquant")
    return t


class AttnLayer:
    """Single-token attention half of a layer (Attention::forward, src/model.rs:79-162, T = 1):
    device-resident Q8_0 weights, RMSNorm weights, rotary tables and the f16 KV cache
    [kv_heads][max_positions][128], with the C struct that points at them."""

    def __init__(self, wq, wk, wv, wo, q_norm, k_norm, rope_cos, rope_sin, hidden: int, query_heads: int = 48,
                 kv_heads: int = 8, rope_dim: int = 64, eps: float = 1e-6):
        import torch
        self.t = (wq, wk, wv, wo, q_norm, k_norm, rope_cos, rope_sin)
        self.max_positions = rope_cos.shape[0]
        self.c = MmrsAttnWeights(wq.data_ptr(), wk.data_ptr(), wv.data_ptr(), wo.data_ptr(), q_norm.data_ptr(),
                                 k_norm.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(), hidden, query_heads,
                                 kv_heads, rope_dim, self.max_positions, eps)
        dev = wq.device
        self.k_cache = torch.zeros(kv_heads, self.max_positions, 128, dtype=torch.float16, device=dev)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.ws = torch.zeros(lib().mmrs_attn_workspace_bytes(C.byref(self.c)), dtype=torch.uint8, device=dev)
        if self.ws.numel() == 0:
            raise MoeError(MMRS_ERR_UNSUPPORTED, "mmrs_attn_workspace_bytes")

    def status(self) -> int:
        """MMRS_OK, or MMRS_ERR_TIMEOUT when a bounded wait in the attention kernel expired."""
        return lib().mmrs_attn_workspace_status(self.ws.data_ptr())

    def forward(self, x, position: int, residual=None, y=None, stream=None):
        """y [hidden] f32 = Wo . attention(x) (+ residual); appends the token's K / V at `position`."""
        import torch
        if y is None:
            y = torch.empty_like(x)
        rc = lib().mmrs_attn_decode_forward(C.byref(self.c), x.data_ptr(), _ptr(residual), position,
                                            self.k_cache.data_ptr(), self.v_cache.data_ptr(), y.data_ptr(),
                                            self.ws.data_ptr(), self.ws.numel(), _stream(stream))
        check(rc, "mmrs_attn_decode_forward")
        return y


class LmHead:
    """Output projection of a decode step (TensorParallelModel::logits, src/tensor_parallel_model.rs:871-880,
    and greedy sampling, src/sampling.rs:84-88): device-resident Q6_K `output.weight` [vocab][hidden]
    and `output_norm.weight` (or None), with the C struct that points at them."""

    def __init__(self, weight, norm_weight, vocab: int, hidden: int, eps: float = 1e-6):
        import torch
        self.t = (weight, norm_weight)
        self.c = MmrsLmHead(weight.data_ptr(), _ptr(norm_weight), vocab, hidden, eps)
        n = lib().mmrs_lm_head_workspace_bytes(C.byref(self.c))
        if n == 0:
            raise MoeError(MMRS_ERR_UNSUPPORTED, "mmrs_lm_head_workspace_bytes")
        self.ws = torch.zeros(n, dtype=torch.uint8, device=weight.device)
        self.logits = torch.empty(vocab, dtype=torch.float32, device=weight.device)
        self.token = torch.zeros(1, dtype=torch.int32, device=weight.device)

    def status(self) -> int:
        return lib().mmrs_lm_head_workspace_status(self.ws.data_ptr())

    def forward(self, x, stream=None):
        """(logits [vocab] f32, token [1] int32) for the final hidden state x [hidden] f32."""
        rc = lib().mmrs_lm_head_forward(C.byref(self.c), x.data_ptr(), self.logits.data_ptr(), self.token.data_ptr(),
                                        self.ws.data_ptr(), self.ws.numel(), _stream(stream))
        check(rc, "mmrs_lm_head_forward")
        return self.logits, self.token


DEFAULT_TEMPERATURE, DEFAULT_TOP_P, DEFAULT_TOP_K = 1.0, 0.95, 40  # src/sampling.rs:6-8


class Sampler:
    """TokenSampler (src/sampling.rs:43-150) over device logits: greedy at temperature 0, else top-k,
    top-p and temperature sampling, the choice made on the device (mmrs_sample_token).  The uniform
    draw is the caller's: `sample(logits, u)` takes it, or draws it from this sampler's own
    generator (numpy PCG64 seeded with `seed`; the reference draws from a per-request StdRng) only
    when the temperature is positive, as the reference draws only then."""

    def __init__(self, vocab: int, device, temperature: float = DEFAULT_TEMPERATURE, top_p: float = DEFAULT_TOP_P,
                 top_k: int = DEFAULT_TOP_K, seed: int = 0):
        import math

        import numpy as np
        import torch
        # SamplingParams::validate (src/sampling.rs:31-39)
        if not math.isfinite(temperature) or temperature < 0.0:
            raise MoeError(MMRS_ERR_ARG, "temperature must be a finite number greater than or equal to 0")
        if not math.isfinite(top_p) or not 0.0 <= top_p <= 1.0:
            raise MoeError(MMRS_ERR_ARG, "top_p must be a finite number between 0 and 1")
        self.params = MmrsSamplingParams(float(temperature), float(top_p), int(top_k))
        self.vocab = vocab
        n = lib().mmrs_sample_workspace_bytes(vocab)
        if n == 0:
            raise MoeError(MMRS_ERR_ARG, "mmrs_sample_workspace_bytes")
        self.ws = torch.zeros(n, dtype=torch.uint8, device=device)
        self.token = torch.full((1,), -1, dtype=torch.int32, device=device)
        self.logprob = torch.zeros(1, dtype=torch.float32, device=device)
        self.rng = np.random.default_rng(seed)

    def status(self) -> int:
        """Outcome of the last completed call (synchronous)."""
        return lib().mmrs_sample_workspace_status(self.ws.data_ptr())

    def sample(self, logits, u: float | None = None, stream=None):
        """token [1] int32 on the device (-1 when status() is not MMRS_OK) for logits [vocab] f32."""
        if u is None:
            u = float(self.rng.random()) if self.params.temperature > 0.0 else 0.0
        rc = lib().mmrs_sample_token(logits.data_ptr(), self.vocab, C.byref(self.params), float(u),
                                     self.token.data_ptr(), self.ws.data_ptr(), self.ws.numel(), _stream(stream))
        check(rc, "mmrs_sample_token")
        return self.token

    def token_logprob(self, logits, token_id: int, stream=None):
        """ln softmax(logits)[token_id] as a [1] f32 device tensor (token_logprob, src/sampling.rs:60-75)."""
        rc = lib().mmrs_token_logprob(logits.data_ptr(), self.vocab, int(token_id), self.logprob.data_ptr(),
                                      self.ws.data_ptr(), self.ws.numel(), _stream(stream))
        check(rc, "mmrs_token_logprob")
        return self.logprob


def rmsnorm(x, weight, y=None, eps: float = 1e-6, stream=None):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last dimension (CUDA f32 tensors)."""
    import torch
    if y is None:
        y = torch.empty_like(x)
    n = x.shape[-1]
    check(lib().mmrs_rmsnorm_f32(x.data_ptr(), weight.data_ptr(), y.data_ptr(), n, x.numel() // n, eps,
                                 _stream(stream)), "mmrs_rmsnorm_f32")
    return y


# ---------------------------------------------------------------------------------------------
# Several sequences: a paged 8-bit cache, attention over it, drafted tokens
# ---------------------------------------------------------------------------------------------
HEAD_DIM = 128  # MMRS_PAGED_HEAD_DIM
PAGE_SIZES = (16, 32, 64, 128)


_TYPE_CODES = {}  # torch dtype -> MMRS_TYPE_* (filled on first use: torch is imported lazily here)


def _type_code(dtype) -> int:
    code = _TYPE_CODES.get(dtype)
    if code is None:
        import torch
        _TYPE_CODES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        code = _TYPE_CODES.get(dtype)
        if code is None:
            raise MoeError(MMRS_ERR_UNSUPPORTED, f"element type {dtype}")
    return code


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise MoeError(MMRS_ERR_ARG, what)


def _on_stream(stream):
    """Where a call allocates: on the stream it runs on, which then owns the memory."""
    import contextlib
    import torch
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _made(t) -> None:
    """Waits until what a constructor wrote is in place: the first call may run on any stream."""
    if t.is_cuda:
        import torch
        torch.cuda.current_stream(t.device).synchronize()


def _same_device(dev: int, *tensors) -> None:
    """The kernels follow raw pointers: every tensor of a call lies on one GPU."""
    if dev < 0:
        raise MoeError(MMRS_ERR_ARG, "tensors on a GPU")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise MoeError(MMRS_ERR_ARG, f"tensors on GPU {dev}")


def _tokens(t, heads, what: str):
    """(tokens, heads, elements between token rows) of t [tokens][heads][128], whose rows are contiguous;
    heads None: as many as t has."""
    try:
        n, h, d = t.shape
        row, head, one = t.stride()
    except ValueError:
        n, h, d, row, head, one = 1, -1, 0, 0, 0, 0
    if n == 0:
        return 0, h, h * HEAD_DIM
    if d != HEAD_DIM or one != 1 or h != (heads or h) or h < 1 or (head != HEAD_DIM and h > 1):
        raise MoeError(MMRS_ERR_ARG, f"{what}: [tokens][{heads or 'heads'}][{HEAD_DIM}], heads side by side")
    return n, h, row if n > 1 else h * HEAD_DIM  # (the stride of a single row is never used and may be anything)


def _on_gpu(dev: int):
    """Makes GPU `dev` the current one.  A kernel is launched on the current GPU whatever its pointers: a call
    for tensors of another one runs inside this."""
    import torch
    return torch.cuda.device(dev)


class PagedBatch:
    """The sequences of one call (MmrsPagedBatch): cu_q int32 [n + 1], seq_len int32 [n] (with the call's
    new tokens) and page_table int32 [n][pages], on the device; max_q and max_len bound the numbers of
    new tokens and the lengths, so that neither is read back."""

    def __init__(self, cu_q, seq_len, page_table, max_q: int, max_len: int, total_q: int | None = None):
        import torch
        n = seq_len.numel()
        for t, name in ((cu_q, "cu_q"), (seq_len, "seq_len"), (page_table, "page_table")):
            _need(t.dtype == torch.int32 and t.is_cuda, f"{name}: int32 on the device")
        _need(cu_q.numel() == n + 1 and cu_q.is_contiguous() and seq_len.is_contiguous(), "cu_q [n + 1], seq_len [n]")
        _need(page_table.dim() == 2 and page_table.shape[0] == n and (page_table.stride(1) == 1 or n == 0),
              "page_table [n][pages]")
        _same_device(seq_len.get_device(), cu_q, page_table)
        self.t = (cu_q, seq_len, page_table)
        self.num_seqs, self.total_q = n, total_q
        # a row stride larger than the row is only ever indexed up to max_len
        self.c = MmrsPagedBatch(cu_q.data_ptr(), seq_len.data_ptr(), page_table.data_ptr(), n,
                                page_table.stride(0) if n > 1 else page_table.shape[1], total_q or 0, max_q, max_len)
        self._ref = C.byref(self.c)
        self._pages = page_table.shape[1]
        self.max_len = max_len

    def bind(self, cache: "PagedKvCache", tokens: int):
        """The C struct for a call with `tokens` token rows."""
        if self._pages * cache.page_size < self.max_len and self.num_seqs:
            raise MoeError(MMRS_ERR_ARG, "page_table: too few pages for max_len")
        if self.total_q is not None and self.total_q != tokens:
            raise MoeError(MMRS_ERR_ARG, "total_q")
        self.c.total_q = tokens
        return self._ref


class PagedKvCache:
    """One layer's keys and values for several sequences, in pages of 16 to 128 positions: e4m3 codes
    [pages][kv_heads][page_size][128] and one f32 scale per page and head (a code's value is code x
    scale).  `append` writes a batch's new tokens, `attend` is the attention of those tokens."""

    def __init__(self, num_pages: int, device, kv_heads: int = 8, page_size: int = 64):
        import torch
        shape = (num_pages, kv_heads, page_size, HEAD_DIM)
        self._bind(*(torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)),
                   *(torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))
        _made(self.k)

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "PagedKvCache":
        """A cache over the caller's own tensors."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale):
        import torch
        _need(k.dim() == 4 and k.shape == v.shape and k.shape[3] == HEAD_DIM and k.dtype == v.dtype ==
              torch.float8_e4m3fn and k.is_contiguous() and v.is_contiguous(),
              "k, v: contiguous float8_e4m3fn [pages][kv_heads][page_size][128]")
        _need(k_scale.shape == v_scale.shape == k.shape[:2] and k_scale.dtype == v_scale.dtype == torch.float32 and
              k_scale.is_contiguous() and v_scale.is_contiguous(), "k_scale, v_scale: f32 [pages][kv_heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device_index = k.get_device()  # -1: no GPU's, which append and attend refuse
        if self.device_index >= 0:
            _same_device(self.device_index, v, k_scale, v_scale)
        pages, self.kv_heads, self.page_size = k.shape[:3]
        if self.page_size not in PAGE_SIZES:
            raise MoeError(MMRS_ERR_UNSUPPORTED, f"page_size {self.page_size}")
        self.c = MmrsPagedCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
                                self.page_size, self.kv_heads)
        self._ref = C.byref(self.c)
        # the GPU that launches go to; the handle of a GPU's current stream (without making a Stream object)
        self._gpu_now, self._raw_now = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        self.ws, self._ws_need = None, {}  # workspace bytes by (sequences, tokens, query heads)
        self._spaces = []  # every workspace handed out: captured graphs go on using the one that they were captured with

    def append(self, batch: PagedBatch, q, k, v, rope_cos, rope_sin, q_out=None, stream=None):
        """Writes the rotated k and v [tokens][kv_heads][128] (f32, f16 or bf16; row slices of one wider
        tensor will do) at the batch's positions; returns the rotated q (bf16 for bf16 queries, else
        f16; None for q None).  rope_cos / rope_sin: f32 [positions][rope_dim / 2]."""
        dtype = k.dtype
        code = _type_code(dtype)
        _same_device(self.device_index, batch.t[1], q, k, v, rope_cos, rope_sin, q_out)
        if self._gpu_now() != self.device_index:
            with _on_gpu(self.device_index):
                return self.append(batch, q, k, v, rope_cos, rope_sin, q_out, stream)
        n, _, k_stride = _tokens(k, self.kv_heads, "k")
        v_n, _, v_stride = _tokens(v, self.kv_heads, "v")
        if v_n != n or v.dtype is not dtype:
            raise MoeError(MMRS_ERR_ARG, "q, k, v: the same tokens, one element type")
        rope, f32 = rope_cos.shape, self.k_scale.dtype
        if (len(rope) != 2 or rope != rope_sin.shape or rope_cos.dtype is not f32 or rope_sin.dtype is not f32 or
                not rope_cos.is_contiguous() or not rope_sin.is_contiguous()):
            raise MoeError(MMRS_ERR_ARG, "rope_cos, rope_sin: f32 [positions][rope_dim / 2]")
        heads = q_stride = out_code = 0
        q_ptr = out_ptr = None
        if q is not None:
            q_n, heads, q_stride = _tokens(q, None, "q")
            if q_n != n or q.dtype is not dtype:
                raise MoeError(MMRS_ERR_ARG, "q, k, v: the same tokens, one element type")
            if q_out is None:
                import torch
                with _on_stream(stream):
                    q_out = torch.empty(n, heads, HEAD_DIM, device=q.device,
                                        dtype=torch.bfloat16 if code == 2 else torch.float16)
            elif q_out.shape != q.shape or not q_out.is_contiguous():
                raise MoeError(MMRS_ERR_ARG, "q_out: contiguous, shaped as q")
            out_code = _type_code(q_out.dtype)
            q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        rc = lib().mmrs_paged_append(self._ref, batch.bind(self, n), q_ptr, k.data_ptr(), v.data_ptr(), q_stride,
                                     k_stride, v_stride, code, heads, rope_cos.data_ptr(), rope_sin.data_ptr(),
                                     2 * rope[1], rope[0], out_ptr, out_code,
                                     self._raw_now(self.device_index) if stream is None else stream.cuda_stream)
        if rc:
            raise MoeError(rc, "mmrs_paged_append")
        return q_out

    def workspace(self, num_seqs: int, tokens: int, query_heads: int, stream=None):
        """The attention's workspace, large enough for such a call; a new one is zeroed on `stream`.  There are two
        sizes (up to 48 rows a KV head, 5 MB, and above, 39 MB); a smaller one stays as long as the cache, for the
        graphs that were captured with it.  None is made inside a capture, where the zeroing would only be
        recorded: call this, or `attend`, for the largest call before it."""
        key = (num_seqs, tokens, query_heads)
        need = self._ws_need.get(key)
        if need is None:
            need = lib().mmrs_paged_attend_workspace_bytes(num_seqs, tokens, query_heads, self.kv_heads)
            if need == 0:
                raise MoeError(MMRS_ERR_UNSUPPORTED, "mmrs_paged_attend_workspace_bytes")
            self._ws_need[key] = need
        if self.ws is None or self.ws.numel() < need:
            import torch
            with _on_stream(stream):
                if self.device_index >= 0 and torch.cuda.is_current_stream_capturing():
                    raise MoeError(MMRS_ERR_ARG, "a workspace cannot be made inside a capture: call workspace() before it")
                self.ws = torch.zeros(need, dtype=torch.uint8, device=self.k.device)
            self._spaces.append(self.ws)
            self._ws_ptr, self._ws_bytes = self.ws.data_ptr(), need
        return self.ws

    def status(self) -> int:
        """MMRS_OK, or MMRS_ERR_TIMEOUT when a bounded wait in an attention kernel expired (synchronous)."""
        return next((st for st in (lib().mmrs_paged_attend_status(w.data_ptr()) for w in self._spaces) if st), MMRS_OK)

    def attend(self, batch: PagedBatch, q, scale: float | None = None, window: int = 0, sinks: int = 0, out=None,
               lse=None, stream=None):
        """out [tokens][heads][128] = attention of q (f16 or bf16, rotated) over the batch's positions up to
        each token's own; with window > 0 only the last `window` of them and the first `sinks`.  lse
        f32 [tokens][heads] is filled when given.  scale: 1 / sqrt(128) unless given.  The calls of
        one cache share a workspace: keep them on one stream.  A captured call needs the cache (which owns the
        workspace) for as long as its graph is replayed, and a call of its size, or `workspace`, before it."""
        n, heads, stride = _tokens(q, None, "q")
        _same_device(self.device_index, batch.t[1], q, out, lse)
        if self._gpu_now() != self.device_index:
            with _on_gpu(self.device_index):
                return self.attend(batch, q, scale, window, sinks, out, lse, stream)
        if out is None:
            import torch
            with _on_stream(stream):
                out = torch.empty(n, heads, HEAD_DIM, dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
            raise MoeError(MMRS_ERR_ARG, "out: contiguous, shaped as q")
        lse_ptr = None
        if lse is not None:
            if lse.shape != (n, heads) or _type_code(lse.dtype) or not lse.is_contiguous():
                raise MoeError(MMRS_ERR_ARG, "lse: f32 [tokens][heads]")
            lse_ptr = lse.data_ptr()
        self.workspace(batch.num_seqs, n, heads, stream)
        rc = lib().mmrs_paged_attend(self._ref, batch.bind(self, n), q.data_ptr(), stride, _type_code(q.dtype), heads,
                                     HEAD_DIM ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(), lse_ptr,
                                     self._ws_ptr, self._ws_bytes,
                                     self._raw_now(self.device_index) if stream is None else stream.cuda_stream)
        if rc:
            raise MoeError(rc, "mmrs_paged_attend")
        return out


class DraftVerifier:
    """Verification of drafted tokens (mmrs_verify_drafts) with this object's outputs and workspace, for up
    to max_seqs sequences of max_q logits rows (drafts + 1) and max_rows rows in all."""

    def __init__(self, vocab: int, device, max_seqs: int, max_rows: int, max_q: int):
        import torch
        need = lib().mmrs_verify_workspace_bytes(max_seqs, max_rows)
        if need == 0 or max_seqs < 1:
            raise MoeError(MMRS_ERR_ARG, "mmrs_verify_workspace_bytes")
        self.vocab, self.max_seqs, self.max_rows, self.max_q = vocab, max_seqs, max_rows, max_q
        # the GPU that launches go to; the handle of a GPU's current stream (without making a Stream object)
        self._gpu_now, self._raw_now = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        self.ws = torch.zeros(need, dtype=torch.uint8, device=device)
        self.tokens = torch.full((max_seqs, max_q), -1, dtype=torch.int32, device=device)
        self.accepted = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.logprobs = torch.zeros(max_seqs, max_q, dtype=torch.float32, device=device)
        _made(self.ws)
        self._ptrs = (self.tokens.data_ptr(), self.accepted.data_ptr(), self.logprobs.data_ptr(), self.ws.data_ptr(), need)

    def status(self) -> int:
        """MMRS_OK, or MMRS_ERR_NONFINITE when some next token of the last call is -1 (synchronous)."""
        return lib().mmrs_verify_workspace_status(self.ws.data_ptr())

    def verify(self, logits, cu_rows, draft_tokens, uniforms, noise, draft_probs=None, temperature=None, stream=None):
        """(tokens [n][max_q] int32, accepted [n] int32, logprobs [n][max_q] f32), valid until the next call:
        the drafts that stand and one more token a sequence, -1 (0.0) after them.  logits [rows][vocab]
        (f32, f16, bf16), cu_rows int32 [n + 1], draft_tokens int32 and uniforms f32 [drafts],
        draft_probs f32 [drafts][vocab] or None (drafts that were certain), noise f32 [n][vocab]
        (exponential), temperature f32 [n] or None (1).  A row whose draft is not among them (sequences without
        rows leave more rows to judge than rows - n) judges none: the next token is drawn there."""
        n, (rows, vocab) = cu_rows.numel() - 1, logits.shape
        drafts = draft_tokens.numel()
        if not 0 <= n <= self.max_seqs or rows > self.max_rows:
            raise MoeError(MMRS_ERR_ARG, "more sequences or rows than the verifier was made for")
        if vocab != self.vocab or not logits.is_contiguous():
            raise MoeError(MMRS_ERR_ARG, "logits [rows][vocab]")
        dev = self.tokens.get_device()
        _same_device(dev, logits, cu_rows, draft_tokens, uniforms, noise, draft_probs, temperature)
        if self._gpu_now() != dev:
            with _on_gpu(dev):
                return self.verify(logits, cu_rows, draft_tokens, uniforms, noise, draft_probs, temperature, stream)
        i32, f32 = self.tokens.dtype, self.logprobs.dtype
        if (cu_rows.dtype != i32 or draft_tokens.dtype != i32 or not cu_rows.is_contiguous() or
                not draft_tokens.is_contiguous()):
            raise MoeError(MMRS_ERR_ARG, "cu_rows, draft_tokens: contiguous int32")
        if uniforms.dtype != f32 or uniforms.numel() != drafts or drafts < rows - n or not uniforms.is_contiguous():
            raise MoeError(MMRS_ERR_ARG, "uniforms f32 [drafts]")
        if noise.dtype != f32 or noise.shape != (n, vocab) or not noise.is_contiguous():
            raise MoeError(MMRS_ERR_ARG, "noise f32 [n][vocab]")
        probs_ptr = temp_ptr = None
        if draft_probs is not None:
            if draft_probs.dtype != f32 or draft_probs.shape != (drafts, vocab) or not draft_probs.is_contiguous():
                raise MoeError(MMRS_ERR_ARG, "draft_probs f32 [drafts][vocab]")
            probs_ptr = draft_probs.data_ptr()
        if temperature is not None:
            if temperature.dtype != f32 or temperature.numel() != n or not temperature.is_contiguous():
                raise MoeError(MMRS_ERR_ARG, "temperature f32 [n]")
            temp_ptr = temperature.data_ptr()
        rc = lib().mmrs_verify_drafts_n(logits.data_ptr(), _type_code(logits.dtype), vocab, cu_rows.data_ptr(), n, rows,
                                        self.max_q, draft_tokens.data_ptr(), probs_ptr, uniforms.data_ptr(), drafts,
                                        noise.data_ptr(), temp_ptr, *self._ptrs,
                                        self._raw_now(dev) if stream is None else stream.cuda_stream)
        if rc:
            raise MoeError(rc, "mmrs_verify_drafts")
        if n == self.max_seqs:
            return self.tokens, self.accepted, self.logprobs
        return self.tokens[:n], self.accepted[:n], self.logprobs[:n]
