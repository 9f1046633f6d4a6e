"""ctypes binding of libfl355.so (include/fl355.h).

The library is loaded once, from this package directory. There is no
fallback: if it is missing or does not load, importing the op layer raises,
so nothing can silently run another implementation. The paged entry points
have a compiled binding as well (fl355_paged.so), which calls the same
library with less work on the host.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import warnings
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libfl355.so"

FL_OK, FL_EINVAL, FL_ELAUNCH, FL_ESCRATCH = 0, 1, 2, 3
FL_MAX_SEQS = 16

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_LL = ctypes.c_longlong
_SZ = ctypes.c_size_t
_PP = ctypes.POINTER(ctypes.c_void_p)
_IP = ctypes.POINTER(ctypes.c_int)

# name -> (restype, argtypes); the order is the header's
SIGNATURES = {
    "fl_abi_version": (_I, []),
    "fl_header_digest": (ctypes.c_char_p, []),
    "fl_strerror": (ctypes.c_char_p, [_I]),
    "fl_last_error": (ctypes.c_char_p, []),
    "fl_kv_store": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P]),
    "fl_rmsnorm1p": (_I, [_P, _P, _P, _I, _I, _I, _I, _F, _P]),
    "fl_rope_partial": (_I, [_P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _P]),
    "fl_attn_prep": (_I, [_P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _F,
                          _P]),
    "fl_attention_split_gqa": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _F, _I,
                                    _I, _I, _P]),
    "fl_attention_merge": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _I, _I, _P]),
    "fl_attn_gate": (_I, [_P, _P, _I, _I, _I, _I, _I, _I, _P]),
    "fl_attn_decode_work_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_attn_decode": (_I, [_P, _I, _PP, _PP, _IP, _IP, _I, _I, _I, _I, _I, _F, _I, _I, _P, _I,
                            _I, _P, _I, _P, _SZ, _P]),
    "fl_attention_prefill": (_I, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _F, _I, _P, _I,
                                  _P]),
    "fl_attn_decode_noalloc": (_I, [_P, _I, _PP, _PP, _IP, _IP, _I, _I, _I, _I, _I, _F, _I, _I,
                                    _P, _I, _I, _P, _I, _P]),
    "fl_attn_decode_noalloc_max_bytes": (_SZ, []),
    "fl_attention_prefill_plan": (_I, [_I, _I, _I, _I, _I, _P, _I]),
    "fl_attention_prefill_pieces": (_I, [_I, _I, _I, _I, _I, _P, _I, _IP, _IP]),
    "fl_attention_prefill_split_count": (_I, [_I, _I, _I, _I]),
    "fl_attention_prefill_split_count_q8": (_I, [_I, _I, _I, _I]),
    "fl_attention_prefill_work_bytes": (_SZ, [_I, _I, _I, _I]),
    "fl_attention_prefill_auto_work_bytes": (_SZ, [_I, _I, _I, _I, _I, _I]),
    "fl_attention_prefill_q8_stage_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_attention_prefill_kv": (_I, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _F, _I, _I,
                                     _P, _I, _P, _SZ, _P]),
    "fl_attention_prefill_kv_q8": (_I, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _F, _I,
                                        _I, _P, _I, _P, _SZ, _P]),
    "fl_attention_prefill_gated": (_I, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _F,
                                        _I, _I, _P, _I, _P, _SZ, _P]),
    "fl_kv_store_q8": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P]),
    "fl_attn_prep_q8": (_I, [_P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F,
                             _F, _P]),
    "fl_attn_prep_rows": (_I, [_P, _I, _P, _P, _P, _P, _PP, _PP, _IP, _IP, _I, _I, _I, _I, _I,
                               _I, _F, _F, _P]),
    "fl_attention_split_gqa_q8": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _F,
                                       _I, _I, _I, _P]),
    "fl_attention_dec_q8": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _F, _I, _I, _I, _P]),
    "fl_attention_dec_merge": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _I, _I, _P]),
    "fl_attn_decode_q8": (_I, [_P, _I, _PP, _PP, _IP, _IP, _I, _I, _I, _I, _I, _F, _I, _I, _P,
                               _I, _I, _P, _I, _P, _SZ, _P]),
    "fl_attention_prefill_q8": (_I, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _F, _I, _P,
                                     _I, _P]),
    "fl_paged_kv_store": (_I, [_P, _P, _LL, _LL, _P, _P, _I, _I, _I, _P, _I, _LL, _P, _P, _I, _I, _I,
                               _I, _P]),
    "fl_paged_kv_load": (_I, [_P, _P, _I, _I, _I, _P, _I, _LL, _P, _P, _P, _P, _LL, _LL, _I, _I, _I,
                              _I, _I, _P]),
    "fl_attn_prep_paged": (_I, [_P, _I, _P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _P, _I, _LL, _P,
                                _P, _I, _I, _I, _I, _I, _I, _F, _F, _P]),
    "fl_attention_prefill_paged_work_bytes": (_SZ, [_IP, _IP, _I, _I, _I, _I, _I, _I, _I]),
    "fl_attention_prefill_paged": (_I, [_P, _I, _P, _P, _I, _I, _I, _P, _I, _LL, _IP, _IP, _I, _I, _I,
                                        _I, _F, _I, _I, _I, _P, _I, _P, _SZ, _P]),
    "fl_attn_decode_paged_work_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_attn_decode_paged": (_I, [_P, _I, _P, _P, _I, _I, _I, _P, _I, _LL, _P, _I, _I, _I, _I, _I, _F,
                                  _I, _I, _I, _P, _I, _P, _SZ, _P]),
    "fl_attn_prep_axes": (_I, [_P, _I, _P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _P, _I, _LL, _P,
                               _P, _P, _I, _IP, _I, _I, _I, _I, _I, _I, _F, _F, _P]),
    "fl_attn_tree_paged_work_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_attn_tree_paged": (_I, [_P, _I, _P, _P, _I, _I, _I, _P, _I, _LL, _P, _P, _I, _I, _I, _I, _I, _F,
                                _I, _I, _I, _P, _I, _P, _SZ, _P]),
    "fl_paged_kv_copy": (_I, [_PP, _PP, _I, _I, _I, _I, _P, _P, _I, _I, _I, _P]),
    "fl_paged_kv_keep": (_I, [_PP, _PP, _I, _I, _I, _I, _P, _I, _LL, _P, _P, _I, _I, _I, _I, _P]),
    "fl_gdn_tree_normed": (_I, [_P, _I, _P, _PP, _IP, _P, _P, _P, _I, _P, _P, _PP, _P, _I, _P, _P,
                                _I, _I, _I, _I, _I, _I, _I, _F, _F, _F, _P]),
    "fl_gdn_tree_commit": (_I, [_P, _I, _P, _PP, _PP, _IP, _P, _P, _P, _I, _P, _P, _PP, _PP, _I, _I,
                                _I, _I, _I, _I, _I, _F, _P]),
    "fl_conv1d_causal": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P]),
    "fl_conv1d_causal_rows": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "fl_l2norm_scaled": (_I, [_P, _P, _I, _I, _I, _F, _F, _I, _P]),
    "fl_l2norm_scaled_strided": (_I, [_P, _P, _I, _I, _LL, _F, _F, _I, _P]),
    "fl_rmsnorm_gated": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _F, _P]),
    "fl_gdn_scalars": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "fl_gdn_scan": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _I, _P,
                         _LL, _P]),
    "fl_gdn_decode": (_I, [_P, _I, _I, _P, _PP, _PP, _IP, _P, _P, _I, _P, _P, _PP, _P, _I, _PP,
                           _LL, _I, _I, _I, _I, _I, _I, _F, _F, _P]),
    "fl_gdn_decode_normed": (_I, [_P, _I, _I, _P, _PP, _PP, _IP, _P, _P, _I, _P, _P, _PP, _PP,
                                  _LL, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _I, _F, _F, _F,
                                  _P]),
    "fl_gdn_verify_normed": (_I, [_P, _I, _P, _P, _P, _P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _LL,
                                  _P, _P, _P, _I, _I, _I, _I, _I, _F, _F, _F, _P, _SZ, _P]),
    "fl_gdn_chunked_work_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_gdn_prefill_chunked": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I,
                                    _F, _I, _I, _P, _SZ, _P]),
    "fl_gdn_prefill_chunked_logits": (_I, [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I,
                                           _I, _I, _I, _I, _I, _F, _I, _I, _P, _SZ, _P]),
    "fl_gdn_prefill_layer_work_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "fl_gdn_prefill_layer": (_I, [_P, _I, _P, _P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _P, _P, _I,
                                  _I, _I, _I, _I, _F, _F, _F, _P, _SZ, _P]),
}


class FlError(RuntimeError):
    """A libfl355 entry point refused its arguments or a launch failed."""

    def __init__(self, fn: str, status: int, detail: str):
        super().__init__(f"{fn}: {detail or 'status %d' % status}")
        self.status = status


_lib = None
# the compiled binding of the paged entry points (csrc/paged_binding.cpp), once the library is
# loaded; None where it has not been built, or for another library or torch: ops.py then makes
# the same calls through ctypes
lane = None
BINDING_PATH = LIB_PATH.with_name("fl355_paged.so")
BOUND = ("fl_paged_kv_store", "fl_paged_kv_load", "fl_attn_prep_paged",
         "fl_attention_prefill_paged_work_bytes", "fl_attention_prefill_paged",
         "fl_attn_decode_paged_work_bytes", "fl_attn_decode_paged", "fl_attn_prep_axes",
         "fl_paged_kv_copy", "fl_paged_kv_keep", "fl_gdn_tree_normed", "fl_gdn_tree_commit",
         "fl_attn_tree_paged_work_bytes", "fl_attn_tree_paged")


def _load_binding(L: ctypes.CDLL, path: Path | None = None):
    path = path or BINDING_PATH
    if not path.exists():
        return None
    loader = importlib.machinery.ExtensionFileLoader("fl355_paged", str(path))
    try:
        module = importlib.util.module_from_spec(
            importlib.util.spec_from_file_location("fl355_paged", path, loader=loader))
        loader.exec_module(module)
    except ImportError:   # (built for another torch)
        return None
    import torch
    built_for, here = getattr(module, "built_for", None), (L.fl_header_digest().decode(), torch.__version__)
    if built_for != here:   # its calls' arguments, or its tensors, may be laid out differently
        warnings.warn(f"{path.name} is not used: built for (header, torch) {built_for}, here are "
                      f"{here}; build again", RuntimeWarning, stacklevel=2)
        return None
    module.bind(*(ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in BOUND))
    return module


def lib() -> ctypes.CDLL:
    """The loaded library (raises if it has not been built)."""
    global _lib, lane
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(hipcc, gfx950); there is no fallback implementation")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        lane = _load_binding(L)
        _lib = L
    return _lib


def call(name: str, *args) -> None:
    """Call an int-returning entry point; raise FlError on a non-zero status."""
    rc = getattr(_lib or lib(), name)(*args)
    if rc != FL_OK:
        fail(name, rc)


def fail(name: str, rc: int) -> None:
    """Raise what an entry point's non-zero status says."""
    detail = lib().fl_last_error().decode(errors="replace")
    if rc == FL_EINVAL:
        raise ValueError(f"{name}: {detail}")
    raise FlError(name, rc, detail)


# array types by length: making one costs more than filling it
_PTRS = [ctypes.c_void_p * max(1, n) for n in range(FL_MAX_SEQS + 1)]
_INTS = [ctypes.c_int * max(1, n) for n in range(FL_MAX_SEQS + 1)]


def ptr_array(ptrs) -> ctypes.Array:
    n = len(ptrs)
    return (_PTRS[n] if n <= FL_MAX_SEQS else ctypes.c_void_p * n)(*ptrs)


def int_array(vals) -> ctypes.Array:
    n = len(vals)
    return (_INTS[n] if n <= FL_MAX_SEQS else ctypes.c_int * n)(*map(int, vals))
