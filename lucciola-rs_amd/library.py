"""ctypes binding of liblucattn.so (include/luc_attn.h) over torch tensors.

torch is imported first so that the library binds to the HIP runtime torch has
already loaded (both name it libamdhip64.so.7): device pointers and streams
from torch are then valid in the library.
"""
from __future__ import annotations

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))

LUC_BF16 = 0
LUC_F16 = 1
STATUS = {0: "LUC_OK", -1: "LUC_E_INVALID", -2: "LUC_E_UNSUPPORTED", -3: "LUC_E_LOAD",
          -4: "LUC_E_HIP", -5: "LUC_E_WORKSPACE", -6: "LUC_E_NOMEM"}

_vp = ctypes.c_void_p
_i32 = ctypes.c_int
_i64 = ctypes.c_int64
_f32 = ctypes.c_float
_sz = ctypes.c_size_t

# name -> (restype, argtypes); every function declared in include/luc_attn.h
SIGNATURES = {
    "luc_abi_version": (_i32, []),
    "luc_last_error": (ctypes.c_char_p, []),
    "luc_init": (_i32, [_i32, ctypes.c_char_p, ctypes.POINTER(_vp)]),
    "luc_destroy": (None, [_vp]),
    "luc_rope_table": (_i32, [_vp, _vp, _i32, _i32, _f32, _f32]),
    "luc_rope": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _i32, _i32, _i32,
                        _i32]),
    "luc_kv_cache_update": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i32, _i32,
                                   _vp, _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_rope_append": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp,
                               _vp, _i32, _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32,
                               _i32]),
    "luc_paged_decode_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_paged_decode": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _i32, _i32,
                                _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _f32, _i32,
                                _vp, _sz]),
    "luc_decode_step": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                               _i32, _i32, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                               _f32, _i32, _vp, _i64, _vp, _sz]),
    "luc_decode_step_noalloc": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp,
                                       _vp, _vp, _i32, _i32, _vp, _i32, _i32, _i32, _i32, _i32,
                                       _i32, _i32, _i32, _f32, _i32, _vp, _i64]),
    "luc_paged_prefill": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                 _vp, _i32, _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32,
                                 _i32, _i32, _i32, _f32, _vp, _i64]),
    "luc_paged_prefill_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_paged_prefill_split": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                       _vp, _i32, _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32,
                                       _i32, _i32, _i32, _f32, _vp, _i64, _vp, _sz]),
    "luc_rmsnorm": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _f32, _i32, _i32]),
    "luc_prompt_gemm": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i32, _i32, _i32]),
    "luc_prompt_mlp_workspace_size": (_sz, [_i32, _i32, _i32]),
    "luc_prompt_mlp": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp, _vp, _i32,
                              _i32, _i32, _vp, _sz]),
    "luc_silu_mul": (_i32, [_vp, _vp, _i32, _vp, _i32, _i32]),
    "luc_gemv": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _i32, _i32]),
    "luc_rmsnorm_gemv": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _f32, _vp, _vp, _i32, _i32]),
    "luc_gate_up_silu": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _f32, _vp, _i32, _i32]),
    "luc_embedding": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i32, _i32, _i32]),
    "luc_argmax": (_i32, [_vp, _vp, _i32, _vp, _i32, _vp]),
    "luc_sort_and_sample": (_i32, [_vp, _vp, _i32, _vp, _i32, _f32, _i32, _f32, _vp, _sz, _vp]),
    "luc_gather_floor": (_i32, [_vp, _vp, _vp, _vp, _vp, _i32, _i32, _vp, _i32, _i32, _i32, _i32,
                                _i32, _i32, _vp]),
    "luc_stream_read": (_i32, [_vp, _vp, _vp, _sz, _vp]),
    "luc_block_extend": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i32, _vp, _vp, _i32, _i32, _vp, _vp,
                                _vp, _vp]),
    "luc_block_truncate": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i32, _vp, _vp, _i32]),
    "luc_qk_norm_rope_append": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp,
                                       _f32, _vp, _vp, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _i64,
                                       _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv4_page_bytes": (_sz, [_i32]),
    "luc_kv4_append": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _f32,
                              _vp, _vp, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _vp, _i64, _vp, _vp,
                              _i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv4_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv4_attention": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _i32, _i32,
                                 _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                 _i32, _f32, _vp, _sz]),
    "luc_kv8_append": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _f32,
                              _vp, _vp, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _i32,
                              _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv8_read": (_i32, [_vp, _vp, _i32, _vp, _vp, _i64, _vp, _i32, _vp, _vp, _vp, _i32, _i32,
                            _i32, _i32, _i32, _i32]),
    "luc_kv8_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv8_attention": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i32,
                                 _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                 _i32, _i32, _f32, _vp, _sz]),
    "luc_kv8_sparse_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32]),
    "luc_kv8_select": (_i32, [_vp, _vp, _i32, _vp, _i32, _i32, _i32, _vp, _i64, _vp, _vp, _vp, _i32,
                              _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                              _vp, _sz]),
    "luc_kv8_sparse_attention": (_i32, [_vp, _vp, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp,
                                        _i32, _i32, _vp, _i32, _vp, _vp, _i32, _i32, _i32, _i32,
                                        _i32, _i32, _i32, _i32, _i32, _f32, _vp, _sz]),
    "luc_blocks_create": (_i32, [_i32, _i32, _i32, ctypes.POINTER(_vp)]),
    "luc_blocks_destroy": (None, [_vp]),
    "luc_blocks_reserve": (_i32, [_vp, _i32, _i32]),
    "luc_blocks_reserve_batch": (_i32, [_vp, _i32, _vp, _vp]),
    "luc_blocks_release": (_i32, [_vp, _i32]),
    "luc_blocks_num_free": (_i32, [_vp]),
    "luc_blocks_num_pages": (_i32, [_vp, _i32]),
    "luc_blocks_table": (_i32, [_vp, _i32, _i32, _vp, _i32]),
}


def lib_dir() -> str:
    """Directory of the gfx950 code objects (and of liblucattn.so)."""
    return os.path.join(_HERE, "lib")


def lib_path() -> str:
    """liblucattn.so in lib/, or LUC_LIB_PATH: another build of the same
    sources (the CPU sanitizer build of sanitize.py)."""
    return os.environ.get("LUC_LIB_PATH") or os.path.join(lib_dir(), "liblucattn.so")


class LucError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"{STATUS.get(code, code)}: {msg}")
        self.code = code


_CDLL = None


def load_cdll() -> ctypes.CDLL:
    """Load liblucattn.so and declare its signatures (no GPU call)."""
    global _CDLL
    if _CDLL is None:
        path = lib_path()
        if not os.path.exists(path):
            raise LucError(-3, f"{path} is not built (run lucciola-rs_amd/build.py)")
        cdll = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(cdll, name)
            fn.restype = res
            fn.argtypes = args
        _CDLL = cdll
    return _CDLL


def dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return LUC_BF16
    if t.dtype == torch.float16:
        return LUC_F16
    raise TypeError(f"unsupported storage dtype {t.dtype}")


def _p(t):
    """Device address of a tensor for a c_void_p argument (argtypes convert the
    int; a c_void_p object per argument would cost more than the launch)."""
    return None if t is None else t.data_ptr()


def pool_pages(pool, num_layers, num_kv_heads, head_dim) -> int:
    """Pages in a K/V pool tensor ([pages][layers][kv heads][16][head_dim], or
    the same elements flat)."""
    if pool.dim() == 5:
        return int(pool.shape[0])
    return int(pool.numel() // (num_layers * num_kv_heads * 16 * head_dim))


def _stream(stream):
    if stream is None:
        # torch.cuda.current_stream().cuda_stream, without the object (0.2 us of a call, not 1.5)
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    return stream.cuda_stream


class LucAttn:
    """One luc_ctx (code objects loaded on one device) and its entry points."""

    def __init__(self, device: int = 0):
        self.lib = load_cdll()
        self.device = device
        self.ctx = ctypes.c_void_p()
        with torch.cuda.device(device):
            rc = self.lib.luc_init(device, lib_dir().encode(), ctypes.byref(self.ctx))
        self._check(rc)

    def close(self):
        if self.ctx:
            self.lib.luc_destroy(self.ctx)
            self.ctx = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        if rc != 0:
            raise LucError(rc, self.lib.luc_last_error().decode())

    # ---- host helpers --------------------------------------------------
    def rope_table(self, max_pos, head_dim, base=1e6, scale_factor=None):
        cos = torch.empty((max_pos, head_dim // 2), dtype=torch.float32)
        sin = torch.empty((max_pos, head_dim // 2), dtype=torch.float32)
        self._check(self.lib.luc_rope_table(_p(cos), _p(sin), max_pos, head_dim, base,
                                            scale_factor or 0.0))
        return cos, sin

    def workspace_size(self, batch, hq, hkv, head_dim, max_ctx, split_tokens=0):
        return self.lib.luc_paged_decode_workspace_size(batch, hq, hkv, head_dim, max_ctx,
                                                        split_tokens)

    # ---- launches ------------------------------------------------------
    def rope(self, q, q_bias, k, k_bias, row_stride, cos, sin, positions, num_tokens, hq, hkv,
             head_dim, stream=None):
        self._check(self.lib.luc_rope(self.ctx, _stream(stream), dtype_code(q), _p(q), _p(q_bias),
                                      _p(k), _p(k_bias), row_stride, _p(cos), _p(sin),
                                      _p(positions), num_tokens, hq, hkv, head_dim))

    def kv_cache_update(self, k_pool, v_pool, k, v, v_bias, row_stride, tables, positions,
                        num_tokens, layer, num_layers, hkv, head_dim, block_size=16,
                        stream=None, num_blocks=None):
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        self._check(self.lib.luc_kv_cache_update(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(k_pool), _p(v_pool), _p(k), _p(v),
            _p(v_bias), row_stride, _p(tables), tables.shape[-1], nb, _p(positions), num_tokens,
            layer, num_layers, hkv, head_dim, block_size))

    def rope_append(self, q, q_bias, k, k_bias, v, v_bias, row_stride, cos, sin, positions,
                    tables, k_pool, v_pool, num_tokens, layer, num_layers, hq, hkv, head_dim,
                    block_size=16, stream=None, num_blocks=None):
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        self._check(self.lib.luc_rope_append(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(q), _p(q_bias), _p(k), _p(k_bias),
            _p(v), _p(v_bias), row_stride, _p(cos), _p(sin), _p(positions), _p(tables),
            tables.shape[-1], nb, _p(k_pool), _p(v_pool), num_tokens, layer, num_layers, hq, hkv,
            head_dim, block_size))

    def paged_decode(self, out, q, k_pool, v_pool, tables, positions, batch, max_ctx, layer,
                     num_layers, hq, hkv, head_dim, sm_scale, split_tokens=0, workspace=None,
                     out_row_stride=None, q_row_stride=None, block_size=16, stream=None,
                     num_blocks=None):
        ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        self._check(self.lib.luc_paged_decode(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(out),
            out_row_stride if out_row_stride is not None else hq * head_dim, _p(q),
            q_row_stride if q_row_stride is not None else hq * head_dim, _p(k_pool), _p(v_pool),
            _p(tables), tables.shape[-1], nb, _p(positions), batch, max_ctx, layer, num_layers, hq,
            hkv, head_dim, block_size, sm_scale, split_tokens, _p(workspace), ws_bytes))


    def decode_step(self, qkv, q_bias, k_bias, v_bias, cos, sin, k_pool, v_pool, tables,
                    positions, batch, max_ctx, layer, num_layers, hq, hkv, head_dim, sm_scale,
                    out, workspace=None, split_tokens=0, qkv_row_stride=None,
                    out_row_stride=None, block_size=16, stream=None, num_blocks=None):
        ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        self._check(self.lib.luc_decode_step(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(qkv),
            qkv_row_stride if qkv_row_stride is not None else (hq + 2 * hkv) * head_dim,
            _p(q_bias), _p(k_bias), _p(v_bias), _p(cos), _p(sin), _p(k_pool), _p(v_pool),
            _p(tables), tables.shape[-1], nb, _p(positions), batch, max_ctx, layer, num_layers, hq, hkv,
            head_dim, block_size, sm_scale, split_tokens, _p(out),
            out_row_stride if out_row_stride is not None else hq * head_dim, _p(workspace),
            ws_bytes))

    def decode_step_noalloc(self, qkv, q_bias, k_bias, v_bias, cos, sin, k_pool, v_pool, tables,
                            positions, batch, max_ctx, layer, num_layers, hq, hkv, head_dim,
                            sm_scale, out, split_tokens=0, qkv_row_stride=None,
                            out_row_stride=None, block_size=16, stream=None, num_blocks=None):
        """luc_decode_step_noalloc: luc_decode_step with the library's fixed
        per-device scratch as its split-K workspace (no workspace argument)."""
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        self._check(self.lib.luc_decode_step_noalloc(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(qkv),
            qkv_row_stride if qkv_row_stride is not None else (hq + 2 * hkv) * head_dim,
            _p(q_bias), _p(k_bias), _p(v_bias), _p(cos), _p(sin), _p(k_pool), _p(v_pool),
            _p(tables), tables.shape[-1], nb, _p(positions), batch, max_ctx, layer, num_layers, hq, hkv,
            head_dim, block_size, sm_scale, split_tokens, _p(out),
            out_row_stride if out_row_stride is not None else hq * head_dim))

    def paged_prefill(self, qkv, q_bias, k_bias, v_bias, cos, sin, k_pool, v_pool, tables,
                      cu_seqlens, start_pos, total_rows, max_ctx, layer, num_layers, hq, hkv,
                      head_dim, sm_scale, out, qkv_row_stride=None, out_row_stride=None,
                      block_size=16, stream=None, num_blocks=None):
        """luc_paged_prefill_split: rope + cache write + causal attention of
        packed prompts (cu_seqlens [B+1], start_pos [B] device int32), with the
        partials of its K splits in a buffer allocated here, on the launch's
        stream."""
        nb = num_blocks if num_blocks is not None else pool_pages(k_pool, num_layers, hkv, head_dim)
        batch = start_pos.shape[0]
        need = self.lib.luc_paged_prefill_workspace_size(batch, total_rows, max_ctx, hq, hkv, head_dim)
        ws = None
        if need:
            if stream is None:
                ws = torch.empty(need, dtype=torch.uint8, device=k_pool.device)
            else:
                with torch.cuda.stream(stream):
                    ws = torch.empty(need, dtype=torch.uint8, device=k_pool.device)
        self._check(self.lib.luc_paged_prefill_split(
            self.ctx, _stream(stream), dtype_code(k_pool), _p(qkv),
            qkv_row_stride if qkv_row_stride is not None else (hq + 2 * hkv) * head_dim,
            _p(q_bias), _p(k_bias), _p(v_bias), _p(cos), _p(sin), _p(k_pool), _p(v_pool),
            _p(tables), tables.shape[-1], nb, _p(cu_seqlens), _p(start_pos), batch,
            total_rows, max_ctx, layer, num_layers, hq, hkv, head_dim, block_size, sm_scale,
            _p(out), out_row_stride if out_row_stride is not None else hq * head_dim, _p(ws), need))

    # ---- the model loop's small kernels ----
    def rmsnorm(self, out, x, weight, eps, stream=None):
        """luc_rmsnorm over the rows of x ([rows, cols] bf16); out may be x."""
        cols = x.shape[-1]
        self._check(self.lib.luc_rmsnorm(self.ctx, _stream(stream), dtype_code(x), _p(out), _p(x),
                                         _p(weight), eps, x.numel() // cols, cols))

    @staticmethod
    def _gemv_shapes(name, y, x, w, residual):
        n, k = w.shape
        if not (w.is_contiguous() and x.is_contiguous() and y.is_contiguous()) or \
                x.numel() != k or y.numel() != n or \
                (residual is not None and (residual.numel() != n or not residual.is_contiguous())):
            raise ValueError(f"{name}: w {tuple(w.shape)}, x {tuple(x.shape)}, y {tuple(y.shape)}: "
                             "want contiguous x [k], y [n] (and residual [n]) for w [n, k]")
        return n, k

    def prompt_gemm(self, y, x, w, stream=None):
        """luc_prompt_gemm: y = x w^T for the rows of x [rows, k] and w [n, k] bf16."""
        rows, k = x.shape
        n = w.shape[0]
        if not (w.is_contiguous() and x.is_contiguous() and y.is_contiguous()) or \
                w.shape[1] != k or tuple(y.shape) != (rows, n):
            raise ValueError(f"prompt_gemm: w {tuple(w.shape)}, x {tuple(x.shape)}, y {tuple(y.shape)}")
        self._check(self.lib.luc_prompt_gemm(self.ctx, _stream(stream), dtype_code(w), _p(y), _p(x),
                                             _p(w), rows, n, k))

    def prompt_mlp(self, h, att, o_w, post_norm, eps, gate_up_w, down_w, next_norm, x, workspace,
                   stream=None):
        """luc_prompt_mlp: a layer's rows h [rows, hidden] (in place) from its
        attention output; x gets the next layer's normed input (next_norm None:
        scratch).  workspace: uint8 of luc_prompt_mlp_workspace_size."""
        rows, hidden = h.shape
        inter = down_w.shape[1]
        if not all(t.is_contiguous() for t in (h, att, o_w, gate_up_w, down_w, x)) or \
                att.shape != h.shape or x.shape != h.shape or tuple(o_w.shape) != (hidden, hidden) or \
                tuple(gate_up_w.shape) != (2 * inter, hidden) or down_w.shape[0] != hidden or \
                post_norm.numel() != hidden or (next_norm is not None and next_norm.numel() != hidden):
            raise ValueError(f"prompt_mlp: h {tuple(h.shape)}, att {tuple(att.shape)}, o_w {tuple(o_w.shape)}, "
                             f"gate_up_w {tuple(gate_up_w.shape)}, down_w {tuple(down_w.shape)}")
        self._check(self.lib.luc_prompt_mlp(
            self.ctx, _stream(stream), dtype_code(h), _p(h), _p(att), _p(o_w), _p(post_norm), eps,
            _p(gate_up_w), _p(down_w), _p(next_norm), _p(x), rows, hidden, inter, _p(workspace),
            workspace.numel()))

    def gemv(self, y, x, w, residual=None, stream=None):
        """luc_gemv: y = x w^T (+ residual) for one row x [k] (or [1, k]) and
        w [n, k] bf16; residual may be y (an in-place residual add)."""
        n, k = self._gemv_shapes("gemv", y, x, w, residual)
        self._check(self.lib.luc_gemv(self.ctx, _stream(stream), dtype_code(w), _p(y), _p(x), _p(w),
                                      _p(residual), n, k))

    def rmsnorm_gemv(self, y, x, norm_weight, eps, w, residual=None, stream=None):
        """luc_rmsnorm_gemv: y = rmsnorm(x) w^T (+ residual), one row x [k]."""
        n, k = self._gemv_shapes("rmsnorm_gemv", y, x, w, residual)
        if norm_weight.numel() != k:
            raise ValueError(f"rmsnorm_gemv: norm weight of {norm_weight.numel()}, k {k}")
        self._check(self.lib.luc_rmsnorm_gemv(self.ctx, _stream(stream), dtype_code(w), _p(y), _p(x),
                                              _p(norm_weight), eps, _p(w), _p(residual), n, k))

    def gate_up_silu(self, act, x, norm_weight, eps, w, stream=None):
        """luc_gate_up_silu: act [I] = silu(g) * u of [g | u] = rmsnorm(x) w^T
        (x itself when norm_weight is None), w [2 I, k] = [gate; up]."""
        two_i, k = w.shape
        if two_i % 2 or not (w.is_contiguous() and x.is_contiguous() and act.is_contiguous()) or \
                x.numel() != k or act.numel() != two_i // 2 or \
                (norm_weight is not None and norm_weight.numel() != k):
            raise ValueError(f"gate_up_silu: w {tuple(w.shape)}, x {tuple(x.shape)}, act {tuple(act.shape)}: "
                             "want contiguous x [k], act [I] for w [2 I, k]")
        self._check(self.lib.luc_gate_up_silu(self.ctx, _stream(stream), dtype_code(w), _p(act), _p(x),
                                              _p(norm_weight), eps, _p(w), two_i // 2, k))

    def silu_mul(self, gate_up, intermediate, stream=None):
        """luc_silu_mul in place on [rows, 2*intermediate] (gate | up) rows."""
        rows = gate_up.numel() // (2 * intermediate)
        self._check(self.lib.luc_silu_mul(self.ctx, _stream(stream), dtype_code(gate_up),
                                          _p(gate_up), rows, intermediate))

    def embedding(self, out, table, ids, stream=None):
        """luc_embedding: out[t] = table[ids[t]] (ids: device int32/uint32)."""
        self._check(self.lib.luc_embedding(self.ctx, _stream(stream), dtype_code(table), _p(out),
                                           _p(table), _p(ids), ids.numel(), table.shape[0],
                                           table.shape[1]))

    # ---- serving over a cache held on the GPU ----
    # (plain checks without loops or keywords: a call of a small batch takes less on the GPU
    # than its checks on the host otherwise would)
    @staticmethod
    def _array(name, t, dtype, dev, least):
        """An operand read as a flat array: contiguous, of `dtype`, on device `dev` (the library's), of
        at least `least` elements."""
        if t.dtype is not dtype or t.get_device() != dev or t.numel() < least or not t.is_contiguous():
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} on {t.device}: want contiguous {dtype} of at "
                             f"least {least} elements on the library's device")
        return t.data_ptr()

    @staticmethod
    def _rows(name, t, width, head_dim, dtype, dev):
        """(rows, row stride) of an operand [rows, width] or [rows, heads, head_dim] whose rows are
        `width` consecutive elements.  One row has no stride: 2^30 stands for any."""
        shape, strides = t.shape, t.stride()
        if t.dtype is not dtype or t.get_device() != dev:
            raise TypeError(f"{name} is {t.dtype} on {t.device}: want {dtype} on the library's device")
        if len(shape) == 2 and shape[1] == width and strides[1] == 1 or \
                len(shape) == 3 and shape[1] * shape[2] == width and strides[1:] == (head_dim, 1) and shape[2] == head_dim:
            return shape[0], strides[0] if shape[0] > 1 else 1 << 30
        raise ValueError(f"{name} {tuple(shape)} with strides {strides}: want rows of {width} consecutive elements")

    def block_extend(self, new_tokens, lens, tables, free_list, state, slots, positions, cu_seqlens,
                     start_pos, stream=None):
        """luc_block_extend: pages, slots and positions for new_tokens[b] more tokens of each
        sequence b.  tables int32 [B, pages]; free_list int32 [num_blocks]; state int32 [4];
        slots int64 and positions int32 of one length, the most rows of the batch; the others
        int32 [B], cu_seqlens [B + 1]."""
        batch, stride = tables.shape
        i32, rows, dev, arr = torch.int32, slots.numel(), self.device, self._array
        blocks = free_list.numel()
        self._check(self.lib.luc_block_extend(
            self.ctx, _stream(stream), batch, arr("new_tokens", new_tokens, i32, dev, batch),
            arr("lens", lens, i32, dev, batch), arr("tables", tables, i32, dev, 0), stride,
            arr("free_list", free_list, i32, dev, 0), arr("state", state, i32, dev, 4), blocks, rows,
            arr("slots", slots, torch.int64, dev, 0), arr("positions", positions, i32, dev, rows),
            arr("cu_seqlens", cu_seqlens, i32, dev, batch + 1), arr("start_pos", start_pos, i32, dev, batch)))

    def block_truncate(self, keep, lens, tables, free_list, state, stream=None):
        """luc_block_truncate: sequence b back to at most keep[b] tokens, its pages behind those
        to the free list."""
        batch, stride = tables.shape
        i32, dev, arr = torch.int32, self.device, self._array
        self._check(self.lib.luc_block_truncate(
            self.ctx, _stream(stream), batch, arr("keep", keep, i32, dev, batch),
            arr("lens", lens, i32, dev, batch), arr("tables", tables, i32, dev, 0), stride,
            arr("free_list", free_list, i32, dev, 0), arr("state", state, i32, dev, 4), free_list.numel()))

    def _append_args(self, q, k, v, cos, sin, positions, slots, hq, hkv, head_dim, q_norm, k_norm, eps,
                     q_bias, k_bias, v_bias, q_out, stream):
        """The arguments that both appends share, from ctx to q_out_stride, and (rows, dtype, device)."""
        dtype, dev, arr, f32 = q.dtype, self.device, self._array, torch.float32
        qw, kw = hq * head_dim, hkv * head_dim
        rows, stride = own = self._rows("q", q, qw, head_dim, dtype, dev)
        if rows and (self._rows("k", k, kw, head_dim, dtype, dev) != own or
                     self._rows("v", v, kw, head_dim, dtype, dev) != own):
            raise ValueError("k's or v's rows and their stride differ from q's")
        o_stride = stride
        if q_out is None:
            q_out = q
        else:
            o_rows, o_stride = self._rows("q_out", q_out, qw, head_dim, dtype, dev)
            if o_rows != rows:
                raise ValueError(f"q_out has {o_rows} rows, q {rows}")
        table = cos.shape
        max_pos = table[0]
        if table[-1] * 2 != head_dim or table != sin.shape:
            raise ValueError(f"rope tables {tuple(table)}, {tuple(sin.shape)}: want [positions, {head_dim // 2}]")
        return [self.ctx, _stream(stream), dtype_code(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), stride,
                q_bias if q_bias is None else arr("q_bias", q_bias, dtype, dev, qw),
                k_bias if k_bias is None else arr("k_bias", k_bias, dtype, dev, kw),
                v_bias if v_bias is None else arr("v_bias", v_bias, dtype, dev, kw),
                q_norm if q_norm is None else arr("q_norm", q_norm, dtype, dev, head_dim),
                k_norm if k_norm is None else arr("k_norm", k_norm, dtype, dev, head_dim), eps,
                arr("cos", cos, f32, dev, 0), arr("sin", sin, f32, dev, 0), max_pos,
                arr("positions", positions, torch.int32, dev, rows), arr("slots", slots, torch.int64, dev, rows),
                rows, q_out.data_ptr(), o_stride], rows, dtype, dev

    def qk_norm_rope_append(self, q, k, v, cos, sin, positions, slots, k_pool, v_pool, layer, num_layers,
                            hq, hkv, head_dim, q_norm=None, k_norm=None, eps=1e-6, q_bias=None,
                            k_bias=None, v_bias=None, q_out=None, k_out=None, block_size=16,
                            stream=None, num_blocks=None):
        """luc_qk_norm_rope_append: bias, head norms, RoPE and the write to `slots` (int64, as
        block_extend gives them) of the rows q [rows, hq * d], k and v [rows, hkv * d] (views with
        one row stride, as those into a qkv tensor); q_out (default: q itself) gets q, k_out, if
        given, k."""
        args, rows, dtype, dev = self._append_args(q, k, v, cos, sin, positions, slots, hq, hkv, head_dim,
                                                   q_norm, k_norm, eps, q_bias, k_bias, v_bias, q_out, stream)
        k_ptr, k_stride = None, 0
        if k_out is not None:
            k_ptr = k_out.data_ptr()
            o_rows, k_stride = self._rows("k_out", k_out, hkv * head_dim, head_dim, dtype, dev)
            if o_rows != rows:
                raise ValueError(f"k_out has {o_rows} rows, q {rows}")
        page = num_layers * hkv * 16 * head_dim
        pages = min(k_pool.numel(), v_pool.numel()) // page if page > 0 else 0
        if num_blocks is not None:
            if num_blocks > pages:
                raise ValueError(f"num_blocks {num_blocks}: the pools hold {pages} pages")
            pages = num_blocks
        self._check(self.lib.luc_qk_norm_rope_append(
            *args, k_ptr, k_stride, self._array("k_pool", k_pool, dtype, dev, 0),
            self._array("v_pool", v_pool, dtype, dev, 0), pages, layer, num_layers, hq, hkv, head_dim, block_size))

    def _kv4_pools(self, k_pool, v_pool, num_layers, hkv, head_dim, num_blocks, dev):
        """(k address, v address, pages) of 4-bit pools: uint8 [pages, layers, kv heads, 10 * head_dim]."""
        shape = k_pool.shape
        if len(shape) != 4 or shape[1:] != (num_layers, hkv, 10 * head_dim) or v_pool.shape != shape:
            raise ValueError(f"4-bit pools {tuple(shape)}, {tuple(v_pool.shape)}: want [pages, {num_layers}, {hkv}, "
                             f"{10 * head_dim}]")
        pages = shape[0]
        if num_blocks is not None:
            if num_blocks > pages:
                raise ValueError(f"num_blocks {num_blocks}: the pools hold {pages} pages")
            pages = num_blocks
        return (self._array("k_pool", k_pool, torch.uint8, dev, 0), self._array("v_pool", v_pool, torch.uint8, dev, 0),
                pages)

    def kv4_append(self, q, k, v, cos, sin, positions, slots, k_pool, v_pool, layer, num_layers, hq, hkv,
                   head_dim, q_norm=None, k_norm=None, eps=1e-6, q_bias=None, k_bias=None, v_bias=None,
                   q_out=None, k_out=None, v_out=None, block_size=16, stream=None, num_blocks=None):
        """luc_kv4_append: qk_norm_rope_append into 4-bit pools (uint8 [pages, layers, kv heads,
        10 * head_dim]); k_out and v_out (with one row stride), if given, get the values that the
        cache holds now."""
        args, rows, dtype, dev = self._append_args(q, k, v, cos, sin, positions, slots, hq, hkv, head_dim,
                                                   q_norm, k_norm, eps, q_bias, k_bias, v_bias, q_out, stream)
        kp, vp, pages = self._kv4_pools(k_pool, v_pool, num_layers, hkv, head_dim, num_blocks, dev)
        o_stride, width = None, hkv * head_dim
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is not None:
                o_rows, st = self._rows(name, t, width, head_dim, dtype, dev)
                if o_rows != rows or o_stride not in (None, st):
                    raise ValueError(f"{name}: {o_rows} rows of stride {st}; q has {rows} rows, k_out and v_out share "
                                     "one stride")
                o_stride = st
        self._check(self.lib.luc_kv4_append(
            *args, None if k_out is None else k_out.data_ptr(), None if v_out is None else v_out.data_ptr(),
            o_stride or 0, kp, vp, pages, layer, num_layers, hq, hkv, head_dim, block_size))

    def kv4_workspace(self, batch, total_rows, max_rows, max_ctx, hq, hkv, head_dim, device=None):
        """A workspace for kv4_attention calls of these sizes, zero-filled on the current stream (None: none
        needed)."""
        need = self.lib.luc_kv4_workspace_size(batch, total_rows, max_rows, max_ctx, hq, hkv, head_dim)
        if need == 0:
            return None
        return torch.zeros(need // 4, dtype=torch.float32,
                           device=device if device is not None else f"cuda:{self.device}")

    def kv4_attention(self, out, q, k_pool, v_pool, tables, start_pos, batch, total_rows, max_rows,
                      max_ctx, layer, num_layers, hq, hkv, head_dim, sm_scale, cu_seqlens=None,
                      workspace=None, block_size=16, stream=None, num_blocks=None):
        """luc_kv4_attention: out and q [rows, hq * d]; start_pos int32 [batch]; cu_seqlens int32
        [batch + 1], or None for one row a sequence; workspace from kv4_workspace."""
        dtype, dev, arr, i32 = q.dtype, self.device, self._array, torch.int32
        rows, q_stride = self._rows("q", q, hq * head_dim, head_dim, dtype, dev)
        o_rows, o_stride = self._rows("out", out, hq * head_dim, head_dim, dtype, dev)
        if rows < total_rows or o_rows < total_rows:
            raise ValueError(f"q and out have {rows} and {o_rows} rows, fewer than total_rows {total_rows}")
        kp, vp, pages = self._kv4_pools(k_pool, v_pool, num_layers, hkv, head_dim, num_blocks, dev)
        stride = tables.shape[-1]
        ws = None if workspace is None else arr("workspace", workspace, workspace.dtype, dev, 0)
        self._check(self.lib.luc_kv4_attention(
            self.ctx, _stream(stream), dtype_code(q), out.data_ptr(), o_stride, q.data_ptr(), q_stride, kp, vp,
            arr("tables", tables, i32, dev, batch * stride), stride, pages,
            cu_seqlens if cu_seqlens is None else arr("cu_seqlens", cu_seqlens, i32, dev, batch + 1),
            arr("start_pos", start_pos, i32, dev, batch), batch, total_rows, max_rows, max_ctx, layer, num_layers,
            hq, hkv, head_dim, block_size, sm_scale, ws,
            0 if ws is None else workspace.numel() * workspace.element_size()))

    def _kv8_pools(self, k_pool, v_pool, scales, num_layers, hkv, head_dim, num_blocks, dev):
        """(k address, v address, scales address, pages) of 8-bit pools: uint8 [pages, layers, kv heads,
        16 * head_dim], scales float32 [pages, layers, kv heads, 2]."""
        shape, u8 = k_pool.shape, torch.uint8
        pages = shape[0] if shape else 0  # (len() of a tensor takes three times as long)
        want = (pages, num_layers, hkv, 16 * head_dim)
        if shape != want or v_pool.shape != want:
            raise ValueError(f"8-bit pools {tuple(shape)}, {tuple(v_pool.shape)}: want {('pages', *want[1:])}")
        if scales.shape != (pages, num_layers, hkv, 2):
            raise ValueError(f"scales {tuple(scales.shape)}: want {(pages, num_layers, hkv, 2)}")
        # (one test for the three: a call of its own for each would cost a fifth of a launch)
        if k_pool.dtype is not u8 or v_pool.dtype is not u8 or scales.dtype is not torch.float32 or \
                k_pool.get_device() != dev or v_pool.get_device() != dev or scales.get_device() != dev or \
                not (k_pool.is_contiguous() and v_pool.is_contiguous() and scales.is_contiguous()):
            for name, x, dtype in (("k_pool", k_pool, u8), ("v_pool", v_pool, u8), ("scales", scales, torch.float32)):
                self._array(name, x, dtype, dev, 0)
        if num_blocks is not None:
            pages = self._pages_of(pages, num_blocks)
        return k_pool.data_ptr(), v_pool.data_ptr(), scales.data_ptr(), pages

    @staticmethod
    def _pages_of(pages, num_blocks):
        if num_blocks is None:
            return pages
        if num_blocks > pages:
            raise ValueError(f"num_blocks {num_blocks}: the pools hold {pages} pages")
        return num_blocks

    def _bounds(self, bounds, pages, num_layers, hkv, head_dim, dev):
        want = (pages, num_layers, hkv, 2, head_dim)
        if bounds.shape != want:
            raise ValueError(f"bounds {tuple(bounds.shape)}: want {want}")
        return self._array("bounds", bounds, torch.uint8, dev, 0)

    def kv8_append(self, q, k, v, cos, sin, positions, slots, k_pool, v_pool, scales, layer, num_layers, hq, hkv,
                   head_dim, bounds=None, q_norm=None, k_norm=None, eps=1e-6, q_bias=None, k_bias=None,
                   v_bias=None, q_out=None, block_size=16, stream=None, num_blocks=None):
        """luc_kv8_append: qk_norm_rope_append into 8-bit pools (uint8 [pages, layers, kv heads, 16 *
        head_dim]) with their scales (float32 [pages, layers, kv heads, 2]) and, if given, key bounds
        (uint8 [pages, layers, kv heads, 2, head_dim]).  Rows in any order, slots distinct."""
        args, rows, dtype, dev = self._append_args(q, k, v, cos, sin, positions, slots, hq, hkv, head_dim,
                                                   q_norm, k_norm, eps, q_bias, k_bias, v_bias, q_out, stream)
        kp, vp, sp, pages = self._kv8_pools(k_pool, v_pool, scales, num_layers, hkv, head_dim, num_blocks, dev)
        bp = bounds if bounds is None else self._bounds(bounds, k_pool.shape[0], num_layers, hkv, head_dim, dev)
        self._check(self.lib.luc_kv8_append(*args, kp, vp, sp, bp, pages, layer, num_layers, hq, hkv, head_dim,
                                            block_size))

    def kv8_read(self, k_out, v_out, slots, k_pool, v_pool, scales, layer, num_layers, hkv, head_dim,
                 block_size=16, stream=None, num_blocks=None):
        """luc_kv8_read: the tokens of `slots` (int64) to k_out and v_out [rows, hkv * d] (with one row stride)."""
        dtype, dev, width = k_out.dtype, self.device, hkv * head_dim
        rows, stride = own = self._rows("k_out", k_out, width, head_dim, dtype, dev)
        if self._rows("v_out", v_out, width, head_dim, dtype, dev) != own:
            raise ValueError("v_out's rows or their stride differ from k_out's")
        kp, vp, sp, pages = self._kv8_pools(k_pool, v_pool, scales, num_layers, hkv, head_dim, num_blocks, dev)
        self._check(self.lib.luc_kv8_read(
            self.ctx, _stream(stream), dtype_code(k_out), k_out.data_ptr(), v_out.data_ptr(), stride,
            self._array("slots", slots, torch.int64, dev, rows), rows, kp, vp, sp, pages, layer, num_layers, hkv,
            head_dim, block_size))

    def _zeros(self, need, device):
        if need == 0:
            return None
        return torch.zeros(need // 4, dtype=torch.float32,
                           device=device if device is not None else f"cuda:{self.device}")

    def kv8_workspace(self, batch, total_rows, max_rows, max_ctx, hq, hkv, head_dim, device=None):
        """A workspace for kv8_attention calls of these sizes, zero-filled on the current stream (None: none
        needed)."""
        return self._zeros(self.lib.luc_kv8_workspace_size(batch, total_rows, max_rows, max_ctx, hq, hkv, head_dim),
                           device)

    def kv8_sparse_workspace(self, batch, max_ctx, budget, hq, hkv, head_dim, device=None):
        """The same for kv8_select and kv8_sparse_attention."""
        return self._zeros(self.lib.luc_kv8_sparse_workspace_size(batch, max_ctx, budget, hq, hkv, head_dim), device)

    def _batch_args(self, tables, start_pos, cu_seqlens, batch, dev):
        i32, stride = torch.int32, tables.shape[-1]
        if tables.dtype is not i32 or start_pos.dtype is not i32 or tables.get_device() != dev or \
                start_pos.get_device() != dev or tables.numel() < batch * stride or start_pos.numel() < batch or \
                not (tables.is_contiguous() and start_pos.is_contiguous()):
            self._array("tables", tables, i32, dev, batch * stride)
            self._array("start_pos", start_pos, i32, dev, batch)
        return (tables.data_ptr(), stride,
                cu_seqlens if cu_seqlens is None else self._array("cu_seqlens", cu_seqlens, i32, dev, batch + 1),
                start_pos.data_ptr())

    def _workspace_args(self, workspace, dev):
        if workspace is None:
            return None, 0
        if workspace.get_device() != dev or not workspace.is_contiguous():
            self._array("workspace", workspace, workspace.dtype, dev, 0)
        return workspace.data_ptr(), workspace.nbytes

    def kv8_attention(self, out, q, k_pool, v_pool, scales, tables, start_pos, batch, total_rows, max_rows,
                      max_ctx, layer, num_layers, hq, hkv, head_dim, sm_scale, cu_seqlens=None,
                      workspace=None, block_size=16, stream=None, num_blocks=None):
        """luc_kv8_attention: kv4_attention over 8-bit pools and their scales; workspace from kv8_workspace."""
        dtype, dev = q.dtype, self.device
        rows, q_stride = self._rows("q", q, hq * head_dim, head_dim, dtype, dev)
        o_rows, o_stride = self._rows("out", out, hq * head_dim, head_dim, dtype, dev)
        if rows < total_rows or o_rows < total_rows:
            raise ValueError(f"q and out have {rows} and {o_rows} rows, fewer than total_rows {total_rows}")
        kp, vp, sp, pages = self._kv8_pools(k_pool, v_pool, scales, num_layers, hkv, head_dim, num_blocks, dev)
        tp, stride, cu, start = self._batch_args(tables, start_pos, cu_seqlens, batch, dev)
        self._check(self.lib.luc_kv8_attention(
            self.ctx, _stream(stream), dtype_code(q), out.data_ptr(), o_stride, q.data_ptr(), q_stride, kp, vp, sp,
            tp, stride, pages, cu, start, batch, total_rows, max_rows, max_ctx, layer, num_layers, hq, hkv, head_dim,
            block_size, sm_scale, *self._workspace_args(workspace, dev)))

    def _chosen(self, pages, batch, hkv, dev):
        """(address, budget) of pages int32 [batch, hkv, budget]."""
        shape = pages.shape
        if len(shape) != 3 or shape[0] != batch or shape[1] != hkv:
            raise ValueError(f"pages {tuple(shape)}: want [{batch}, {hkv}, budget]")
        return self._array("pages", pages, torch.int32, dev, 0), shape[2]

    def kv8_select(self, pages, q, bounds, scales, tables, start_pos, batch, max_ctx, first, recent, layer,
                   num_layers, hq, hkv, head_dim, cu_seqlens=None, workspace=None, block_size=16, stream=None,
                   num_blocks=None):
        """luc_kv8_select: into pages (int32 [batch, hkv, budget]) the pages that the rows q [rows, hq * d], at most
        one a sequence, attend to; bounds and scales of the pools; workspace from kv8_sparse_workspace."""
        dev = self.device
        rows, q_stride = self._rows("q", q, hq * head_dim, head_dim, q.dtype, dev)
        if cu_seqlens is None and rows < batch:
            raise ValueError(f"q has {rows} rows, fewer than the batch's {batch}")
        shape = scales.shape
        blocks = shape[0] if shape else 0
        if shape != (blocks, num_layers, hkv, 2):
            raise ValueError(f"scales {tuple(shape)}: want [pages, {num_layers}, {hkv}, 2]")
        bp = self._bounds(bounds, blocks, num_layers, hkv, head_dim, dev)
        sp = self._array("scales", scales, torch.float32, dev, 0)
        cp, budget = self._chosen(pages, batch, hkv, dev)
        tp, stride, cu, start = self._batch_args(tables, start_pos, cu_seqlens, batch, dev)
        self._check(self.lib.luc_kv8_select(
            self.ctx, _stream(stream), dtype_code(q), cp, budget, first, recent, q.data_ptr(), q_stride, bp, sp, tp,
            stride, self._pages_of(blocks, num_blocks), cu, start, batch,
            batch if cu_seqlens is None else rows, max_ctx, layer, num_layers, hq, hkv, head_dim, block_size,
            *self._workspace_args(workspace, dev)))

    def kv8_sparse_attention(self, out, q, k_pool, v_pool, scales, tables, start_pos, pages, batch, max_ctx, layer,
                             num_layers, hq, hkv, head_dim, sm_scale, cu_seqlens=None, workspace=None,
                             block_size=16, stream=None, num_blocks=None):
        """luc_kv8_sparse_attention: attention of out and q's rows, at most one a sequence, over the pages that
        kv8_select wrote."""
        dtype, dev = q.dtype, self.device
        rows, q_stride = self._rows("q", q, hq * head_dim, head_dim, dtype, dev)
        o_rows, o_stride = self._rows("out", out, hq * head_dim, head_dim, dtype, dev)
        if o_rows < rows or cu_seqlens is None and rows < batch:
            raise ValueError(f"q and out have {rows} and {o_rows} rows for a batch of {batch}")
        kp, vp, sp, blocks = self._kv8_pools(k_pool, v_pool, scales, num_layers, hkv, head_dim, num_blocks, dev)
        cp, budget = self._chosen(pages, batch, hkv, dev)
        tp, stride, cu, start = self._batch_args(tables, start_pos, cu_seqlens, batch, dev)
        self._check(self.lib.luc_kv8_sparse_attention(
            self.ctx, _stream(stream), dtype_code(q), out.data_ptr(), o_stride, q.data_ptr(), q_stride, kp, vp, sp,
            tp, stride, blocks, cp, budget, cu, start, batch, batch if cu_seqlens is None else rows, max_ctx, layer,
            num_layers, hq, hkv, head_dim, block_size, sm_scale, *self._workspace_args(workspace, dev)))

    def gather_floor(self, k_pool, v_pool, tables, positions, batch, max_ctx, layer, num_layers,
                     hkv, head_dim, sink, stream=None):
        """luc_gather_floor: the decode step's K/V page slabs read with its work
        split and no arithmetic (sink: a one-element device int32 tensor)."""
        self._check(self.lib.luc_gather_floor(
            self.ctx, _stream(stream), _p(k_pool), _p(v_pool), _p(tables), tables.shape[-1],
            pool_pages(k_pool, num_layers, hkv, head_dim), _p(positions), batch, max_ctx, layer,
            num_layers, hkv, head_dim, _p(sink)))

    def stream_read(self, src, sink, stream=None):
        """luc_stream_read of the whole of src (a contiguous device tensor)."""
        self._check(self.lib.luc_stream_read(self.ctx, _stream(stream), _p(src),
                                             src.numel() * src.element_size(), _p(sink)))

    def argmax(self, logits, out_idx, stream=None):
        """luc_argmax into out_idx (a one-element device int32 tensor)."""
        self._check(self.lib.luc_argmax(self.ctx, _stream(stream), dtype_code(logits), _p(logits),
                                        logits.numel(), _p(out_idx)))

    def sort_and_sample(self, logits, top_p, top_k, rand_val, sort_buffer, out_idx, stream=None):
        """luc_sort_and_sample of one bf16 logits row into out_idx (one-element
        device int32 tensor, left unwritten when no candidate is drawn);
        sort_buffer (>= 8*top_k bytes of device memory) returns the sorted
        (index, value) candidates."""
        self._check(self.lib.luc_sort_and_sample(
            self.ctx, _stream(stream), dtype_code(logits), _p(logits), logits.numel(), float(top_p),
            int(top_k), float(rand_val), _p(sort_buffer),
            sort_buffer.numel() * sort_buffer.element_size(), _p(out_idx)))

    def workspace(self, batch, hq, hkv, head_dim, max_ctx, split_tokens=0, device=None):
        """A zero-filled decode workspace (None when no split-K is needed)."""
        need = self.workspace_size(batch, hq, hkv, head_dim, max_ctx, split_tokens)
        if need == 0:
            return None
        return torch.zeros(need // 4, dtype=torch.float32,
                           device=device if device is not None else f"cuda:{self.device}")


_DEFAULT = {}


def default(device: int = 0) -> LucAttn:
    """Process-wide LucAttn for `device` (created on first use)."""
    if device not in _DEFAULT:
        _DEFAULT[device] = LucAttn(device)
    return _DEFAULT[device]
