"""ctypes binding of libmi_hip_attn.so (the C ABI of include/mi_hip_attn.h).

This is a thin test/benchmark front end: the product is the C ABI itself.
Device memory comes from torch (torch.cuda tensors on ROCm); only raw device
addresses cross into the library. Loading fails loudly when the library has
not been built -- there is no fallback path.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmi_hip_attn.so")

MI_TYPE_F32 = 0
MI_TYPE_F16 = 1
MI_TYPE_Q8_0 = 2
MI_TYPE_Q8_0_ACT = 4
MI_HIP_TYPE_Q8 = 100  # cache elements only

MI_OP_NONE = 0
MI_OP_MUL_MAT = 5
MI_OP_ROPE = 6
MI_OP_SOFTMAX = 7
MI_OP_CPY = 10
MI_OP_QUANTIZE_Q8_0 = 11
MI_OP_VIEW = 13
MI_OP_ATTN_QK = 16
MI_OP_ATTN_KQV = 17

MI_TENSOR_FLAG_KV = 1 << 3

MI_HIP_PREFILL_F32 = 0
MI_HIP_PREFILL_SPLIT_BF16 = 1
MI_HIP_PREFILL_AUTO = 2
MI_HIP_DECODE_VALU = 0
MI_HIP_DECODE_MATRIX = 1
MI_HIP_DECODE_AUTO = 2
MI_HIP_DECODE_STREAM = 3

MI_HIP_QWEN2_ATTN_FUSED = 0
MI_HIP_QWEN2_ATTN_REFERENCE_ORDER = 1

STATUS = {0: "OK", 1: "E_INVALID", 2: "E_NODEVICE", 3: "E_RUNTIME", 4: "E_NOMEM",
          5: "E_UNSUPPORTED", 6: "E_STATE", 7: "E_LOST"}


class MiHipError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"{STATUS.get(code, code)}: {msg}")
        self.code = code


class KvHandle(int):
    """A cache handle that knows the shape of the cache's rows."""

    def __new__(cls, handle, n_head_kv, head_dim):
        self = super().__new__(cls, handle)
        self.rows = (n_head_kv, head_dim)
        return self


class MiTensor(ctypes.Structure):
    """ABI mirror of struct mi_tensor (src/tensor.h:122-160)."""


MiTensor._fields_ = [
    ("type", ctypes.c_int),
    ("ne", ctypes.c_int64 * 4),
    ("nb", ctypes.c_size_t * 4),
    ("op", ctypes.c_int),
    ("op_params", ctypes.c_int32 * 8),
    ("src", ctypes.POINTER(MiTensor) * 2),
    ("data", ctypes.c_void_p),
    ("view_src", ctypes.POINTER(MiTensor)),
    ("view_offs", ctypes.c_size_t),
    ("n_children", ctypes.c_int32),
    ("flags", ctypes.c_uint32),
    ("name", ctypes.c_char * 64),
    ("extra", ctypes.c_void_p),
]


class MiCgraph(ctypes.Structure):
    _fields_ = [
        ("nodes", ctypes.POINTER(ctypes.POINTER(MiTensor))),
        ("n_nodes", ctypes.c_int),
        ("leafs", ctypes.POINTER(ctypes.POINTER(MiTensor))),
        ("n_leafs", ctypes.c_int),
        ("exec_nodes", ctypes.POINTER(ctypes.POINTER(MiTensor))),
        ("n_exec_nodes", ctypes.c_int),
        ("capacity", ctypes.c_int),
    ]


class KvDesc(ctypes.Structure):
    _fields_ = [("n_layer", ctypes.c_int32), ("n_ctx", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("n_head", ctypes.c_int32), ("type", ctypes.c_int32)]


class WorkspaceDesc(ctypes.Structure):
    _fields_ = [("n_head_kv", ctypes.c_int32), ("n_head", ctypes.c_int32),
                ("head_dim", ctypes.c_int32)]


class WorkspaceStatus(ctypes.Structure):
    _fields_ = [("early_fallbacks", ctypes.c_uint32), ("lost_groups", ctypes.c_uint32)]


class AttnArgs(ctypes.Structure):
    _fields_ = [
        ("kv", ctypes.c_void_p),
        ("layer", ctypes.c_int32),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_nb", ctypes.c_size_t * 3),
        ("v_nb", ctypes.c_size_t * 3),
        ("kv_type", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("n_head_kv", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("q_nb", ctypes.c_size_t * 3),
        ("out", ctypes.c_void_p),
        ("out_nb", ctypes.c_size_t * 3),
        ("n_head", ctypes.c_int32),
        ("n_rep", ctypes.c_int32),
        ("n_past", ctypes.c_int32),
        ("n_tokens", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("stream", ctypes.c_void_p),
        ("ws", ctypes.c_void_p),
    ]


class RopeArgs(ctypes.Structure):
    _fields_ = [
        ("kv", ctypes.c_void_p),
        ("layer", ctypes.c_int32),
        ("n_past", ctypes.c_int32),
        ("n_tokens", ctypes.c_int32),
        ("n_dims", ctypes.c_int32),
        ("freq_base", ctypes.c_float),
        ("n_head", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("q_nb", ctypes.c_size_t * 3),
        ("q_out", ctypes.c_void_p),
        ("q_out_nb", ctypes.c_size_t * 3),
        ("k", ctypes.c_void_p),
        ("k_nb", ctypes.c_size_t * 3),
        ("v", ctypes.c_void_p),
        ("v_nb", ctypes.c_size_t * 3),
        ("stream", ctypes.c_void_p),
    ]


class NormRopeArgs(ctypes.Structure):
    _fields_ = [
        ("kv", ctypes.c_void_p),
        ("layer", ctypes.c_int32),
        ("n_past", ctypes.c_int32),
        ("n_tokens", ctypes.c_int32),
        ("n_dims", ctypes.c_int32),
        ("freq_base", ctypes.c_float),
        ("freq", ctypes.POINTER(ctypes.c_float)),
        ("pos", ctypes.c_void_p),
        ("eps", ctypes.c_float),
        ("q_norm", ctypes.c_void_p),
        ("k_norm", ctypes.c_void_p),
        ("n_head", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("q_nb", ctypes.c_size_t * 3),
        ("q_out", ctypes.c_void_p),
        ("q_out_nb", ctypes.c_size_t * 3),
        ("k", ctypes.c_void_p),
        ("k_nb", ctypes.c_size_t * 3),
        ("v", ctypes.c_void_p),
        ("v_nb", ctypes.c_size_t * 3),
        ("stream", ctypes.c_void_p),
    ]


class TreeMask(ctypes.Structure):
    _fields_ = [("bits", ctypes.c_void_p), ("nb", ctypes.c_size_t)]


class LogitsArgs(ctypes.Structure):
    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("nb", ctypes.c_size_t),
        ("out", ctypes.c_void_p),
        ("out_nb", ctypes.c_size_t),
        ("n_vocab", ctypes.c_int32),
        ("n_rows", ctypes.c_int32),
        ("penalties", ctypes.c_void_p),
        ("hist", ctypes.c_void_p),
        ("hist_off", ctypes.c_void_p),
        ("bias_id", ctypes.c_void_p),
        ("bias", ctypes.c_void_p),
        ("bias_off", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("mask_nb", ctypes.c_size_t),
        ("ids", ctypes.c_void_p),
        ("ws", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class PageTablesArgs(ctypes.Structure):
    _fields_ = [
        ("n_seq", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("n_pages", ctypes.c_int32),
        ("max_pages", ctypes.c_int32),
        ("max_tokens", ctypes.c_int32),
        ("n_cached", ctypes.c_void_p),
        ("n_new", ctypes.c_void_p),
        ("held", ctypes.c_void_p),
        ("held_out", ctypes.c_void_p),
        ("table", ctypes.c_void_p),
        ("table_nb", ctypes.c_size_t),
        ("ring", ctypes.c_void_p),
        ("ring_at", ctypes.c_void_p),
        ("ring_at_out", ctypes.c_void_p),
        ("n_kv", ctypes.c_void_p),
        ("q_off", ctypes.c_void_p),
        ("slots", ctypes.c_void_p),
        ("pos", ctypes.c_void_p),
        ("seq", ctypes.c_void_p),
        ("n_refused", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class PagedAppendArgs(ctypes.Structure):
    _fields_ = [
        ("kv", ctypes.c_void_p),
        ("layer", ctypes.c_int32),
        ("n_tokens", ctypes.c_int32),
        ("slots", ctypes.c_void_p),
        ("n_dims", ctypes.c_int32),
        ("freq_base", ctypes.c_float),
        ("freq", ctypes.POINTER(ctypes.c_float)),
        ("pos", ctypes.c_void_p),
        ("pos_nb", ctypes.c_size_t),
        ("n_axes", ctypes.c_int32),
        ("axis", ctypes.POINTER(ctypes.c_int32)),
        ("eps", ctypes.c_float),
        ("q_norm", ctypes.c_void_p),
        ("k_norm", ctypes.c_void_p),
        ("n_head", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("q_nb", ctypes.c_size_t * 3),
        ("q_out", ctypes.c_void_p),
        ("q_out_nb", ctypes.c_size_t * 3),
        ("k", ctypes.c_void_p),
        ("k_nb", ctypes.c_size_t * 3),
        ("v", ctypes.c_void_p),
        ("v_nb", ctypes.c_size_t * 3),
        ("stream", ctypes.c_void_p),
    ]


class AttnPagedArgs(ctypes.Structure):
    _fields_ = [
        ("kv", ctypes.c_void_p),
        ("layer", ctypes.c_int32),
        ("n_seq", ctypes.c_int32),
        ("n_tokens", ctypes.c_int32),
        ("max_new", ctypes.c_int32),
        ("q_off", ctypes.c_void_p),
        ("n_kv", ctypes.c_void_p),
        ("table", ctypes.c_void_p),
        ("table_nb", ctypes.c_size_t),
        ("max_pages", ctypes.c_int32),
        ("n_head", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("q_nb", ctypes.c_size_t * 3),
        ("out", ctypes.c_void_p),
        ("out_nb", ctypes.c_size_t * 3),
        ("scale", ctypes.c_float),
        ("ws", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class VerifyArgs(ctypes.Structure):
    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("nb", ctypes.c_size_t),
        ("n_vocab", ctypes.c_int32),
        ("n_rows", ctypes.c_int32),
        ("n_seq", ctypes.c_int32),
        ("off", ctypes.c_void_p),
        ("token", ctypes.c_void_p),
        ("parent", ctypes.c_void_p),
        ("draft", ctypes.c_void_p),
        ("draft_nb", ctypes.c_size_t),
        ("temperature", ctypes.c_void_p),
        ("u", ctypes.c_void_p),
        ("max_path", ctypes.c_int32),
        ("n_path", ctypes.c_void_p),
        ("path", ctypes.c_void_p),
        ("path_nb", ctypes.c_size_t),
        ("tokens", ctypes.c_void_p),
        ("tokens_nb", ctypes.c_size_t),
        ("ws", ctypes.c_void_p),
        ("stream", ctypes.c_void_p),
    ]


class Qwen2Hparams(ctypes.Structure):
    """ABI mirror of mi_hip_qwen2_hparams (include/mi_hip_qwen2.h)."""
    _fields_ = [("n_vocab", ctypes.c_int32), ("n_embd", ctypes.c_int32),
                ("n_layer", ctypes.c_int32), ("n_head", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("n_ff", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("n_ctx_train", ctypes.c_int32),
                ("rope_freq_base", ctypes.c_float), ("rms_eps", ctypes.c_float)]


class AllocStats(ctypes.Structure):
    _fields_ = [("n_malloc", ctypes.c_uint64), ("n_free", ctypes.c_uint64),
                ("bytes_live", ctypes.c_uint64), ("bytes_peak", ctypes.c_uint64)]


_Strides = ctypes.c_size_t * 3


# Every symbol include/mi_hip_attn.h and include/mi_hip_qwen2.h declare, with
# its ctypes signature.
_P = ctypes.c_void_p
_I = ctypes.c_int
SIGNATURES = {
    "mi_hip_init": ([_I], _I),
    "mi_hip_shutdown": ([], _I),
    "mi_hip_last_error": ([], ctypes.c_char_p),
    "mi_hip_abi_layout": ([ctypes.POINTER(ctypes.c_size_t), _I], _I),
    "mi_hip_get_alloc_stats": ([ctypes.POINTER(AllocStats)], _I),
    "mi_hip_set_alloc_limit": ([ctypes.c_uint64], _I),
    "mi_hip_kv_create": ([ctypes.POINTER(KvDesc), ctypes.POINTER(ctypes.c_void_p)], _I),
    "mi_hip_kv_destroy": ([_P], _I),
    "mi_hip_kv_workspace": ([_P, ctypes.POINTER(ctypes.c_void_p)], _I),
    "mi_hip_workspace_create": ([ctypes.POINTER(WorkspaceDesc), ctypes.POINTER(ctypes.c_void_p)], _I),
    "mi_hip_workspace_destroy": ([_P], _I),
    "mi_hip_workspace_check": ([_P, _P, ctypes.POINTER(WorkspaceStatus)], _I),
    "mi_hip_workspace_set_poll_limit": ([_P, ctypes.c_int32], _I),
    "mi_hip_set_deterministic": ([ctypes.c_int32], _I),
    "mi_hip_set_prefill_mode": ([ctypes.c_int32], _I),
    "mi_hip_set_decode_mode": ([ctypes.c_int32], _I),
    "mi_hip_set_host_nodes": ([ctypes.c_int32], _I),
    "mi_hip_decode_tuning": ([ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32], _I),
    "mi_hip_kv_view": ([_P, _I, _I, ctypes.POINTER(ctypes.c_void_p),
                        ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_size_t)], _I),
    "mi_hip_kv_write": ([_P, _I, _I, _I, _I, _P, ctypes.POINTER(ctypes.c_size_t), _I, _P], _I),
    "mi_hip_kv_scales": ([_P, _I, _I, ctypes.POINTER(ctypes.c_void_p),
                          ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_size_t)], _I),
    "mi_hip_kv_read": ([_P, _I, _I, _I, _I, _P, _I, ctypes.POINTER(ctypes.c_size_t), _P], _I),
    "mi_hip_kv_keep": ([_P, _I, _P, _I, _P], _I),
    "mi_hip_kv_bind": ([_P, _I, _I, ctypes.POINTER(MiTensor)], _I),
    "mi_hip_attn_fwd": ([ctypes.POINTER(AttnArgs)], _I),
    "mi_hip_attn_fwd_reference_order": ([ctypes.POINTER(AttnArgs)], _I),
    "mi_hip_attn_decode_batch": ([ctypes.POINTER(AttnArgs), _I, _P], _I),
    "mi_hip_attn_decode_batch_noalloc": ([ctypes.POINTER(AttnArgs), _I, _P], _I),
    "mi_hip_attn_tree": ([ctypes.POINTER(AttnArgs), ctypes.POINTER(TreeMask), _I, _P], _I),
    "mi_hip_op_attn_qk": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_softmax": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_attn_kqv": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_attn_fused": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_rope": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_quantize_q8_0": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_op_mul_mat": ([ctypes.POINTER(MiTensor), _P], _I),
    "mi_hip_rope_append": ([ctypes.POINTER(RopeArgs)], _I),
    "mi_hip_norm_rope_append": ([ctypes.POINTER(NormRopeArgs)], _I),
    "mi_hip_logits_adjust": ([ctypes.POINTER(LogitsArgs)], _I),
    "mi_hip_kv_create_paged": ([ctypes.POINTER(KvDesc), ctypes.c_int32, ctypes.POINTER(ctypes.c_void_p)], _I),
    "mi_hip_page_tables": ([ctypes.POINTER(PageTablesArgs)], _I),
    "mi_hip_paged_append": ([ctypes.POINTER(PagedAppendArgs)], _I),
    "mi_hip_attn_paged": ([ctypes.POINTER(AttnPagedArgs)], _I),
    "mi_hip_verify_draft": ([ctypes.POINTER(VerifyArgs)], _I),
    "mi_hip_memread": ([_P, ctypes.c_size_t, _P, ctypes.c_int32, _P], _I),
    "mi_hip_graph_prepare": ([ctypes.POINTER(MiCgraph)], _I),
    "mi_hip_compute_forward": ([ctypes.POINTER(MiTensor), _I, _I], _I),
    "mi_hip_qwen2_load": ([ctypes.c_char_p, ctypes.c_int32, ctypes.c_int32,
                           ctypes.POINTER(ctypes.c_void_p)], _I),
    "mi_hip_qwen2_free": ([_P], _I),
    "mi_hip_qwen2_get_hparams": ([_P, ctypes.POINTER(Qwen2Hparams)], _I),
    "mi_hip_qwen2_forward": ([_P, ctypes.POINTER(ctypes.c_int32), ctypes.c_int32, ctypes.c_int32,
                              ctypes.c_int32, ctypes.POINTER(ctypes.c_float),
                              ctypes.POINTER(ctypes.c_int32)], _I),
    "mi_hip_qwen2_generate": ([_P, ctypes.POINTER(ctypes.c_int32), ctypes.c_int32, ctypes.c_int32,
                               ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int32)], _I),
    "mi_hip_qwen2_set_attention": ([_P, ctypes.c_int32], _I),
    "mi_hip_qwen2_set_timing": ([_P, ctypes.c_int32], _I),
    "mi_hip_qwen2_get_timing": ([_P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double),
                                 ctypes.POINTER(ctypes.c_int64)], _I),
}


class Lib:
    def __init__(self, path=LIB_PATH):
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is not built: run `make -C mini-infer-llama.cpp_amd` "
                               "(or __graft_entry__.build())")
        self.path = path
        self.so = ctypes.CDLL(path)
        for name, (argtypes, restype) in SIGNATURES.items():
            fn = getattr(self.so, name)
            fn.argtypes = argtypes
            fn.restype = restype

    def last_error(self):
        return self.so.mi_hip_last_error().decode()

    def check(self, rc):
        if rc != 0:
            raise MiHipError(rc, self.last_error())
        return rc

    def __getattr__(self, name):
        return getattr(self.so, name)

    # -- convenience wrappers -------------------------------------------------
    def init(self, device=0):
        self.check(self.so.mi_hip_init(device))

    def alloc_stats(self):
        s = AllocStats()
        self.check(self.so.mi_hip_get_alloc_stats(ctypes.byref(s)))
        return s

    def abi_layout(self):
        arr = (ctypes.c_size_t * 15)()
        self.check(self.so.mi_hip_abi_layout(arr, 15))
        return list(arr)

    def kv_create(self, n_layer, n_ctx, n_head_kv, head_dim, n_head, kv_type=MI_TYPE_F32):
        d = KvDesc(n_layer, n_ctx, n_head_kv, head_dim, n_head, kv_type)
        h = ctypes.c_void_p()
        self.check(self.so.mi_hip_kv_create(ctypes.byref(d), ctypes.byref(h)))
        return KvHandle(h.value, n_head_kv, head_dim)

    def kv_create_paged(self, n_layer, n_pages, page_size, n_head_kv, head_dim, n_head, kv_type=MI_TYPE_F32):
        d = KvDesc(n_layer, n_pages * page_size, n_head_kv, head_dim, n_head, kv_type)
        h = ctypes.c_void_p()
        self.check(self.so.mi_hip_kv_create_paged(ctypes.byref(d), page_size, ctypes.byref(h)))
        return KvHandle(h.value, n_head_kv, head_dim)

    def workspace_create(self, n_head_kv, n_head, head_dim):
        d = WorkspaceDesc(n_head_kv, n_head, head_dim)
        h = ctypes.c_void_p()
        self.check(self.so.mi_hip_workspace_create(ctypes.byref(d), ctypes.byref(h)))
        return h.value

    def kv_workspace(self, kv):
        h = ctypes.c_void_p()
        self.check(self.so.mi_hip_kv_workspace(kv, ctypes.byref(h)))
        return h.value

    def workspace_check(self, ws, stream):
        """(status code, early_fallbacks, lost_groups) since the last check."""
        st = WorkspaceStatus()
        rc = self.so.mi_hip_workspace_check(ws, stream, ctypes.byref(st))
        return rc, st.early_fallbacks, st.lost_groups

    def kv_view(self, kv, layer, which):
        data = ctypes.c_void_p()
        ne = (ctypes.c_int64 * 4)()
        nb = (ctypes.c_size_t * 4)()
        self.check(self.so.mi_hip_kv_view(kv, layer, which, ctypes.byref(data), ne, nb))
        return data.value, list(ne), list(nb)

    def kv_scales(self, kv, layer, which):
        data = ctypes.c_void_p()
        ne = (ctypes.c_int64 * 4)()
        nb = (ctypes.c_size_t * 4)()
        self.check(self.so.mi_hip_kv_scales(kv, layer, which, ctypes.byref(data), ne, nb))
        return data.value, list(ne), list(nb)

    def kv_write(self, kv, layer, which, pos0, src, stream):
        """Rows of an F32 device tensor (n_tokens, n_head_kv, head_dim) into K (which 0) or V (1)."""
        _expect(_kind(src) == MI_TYPE_F32, "src: float32")
        n, nb = _cache_rows(kv, src, 4)
        self.check(self.so.mi_hip_kv_write(kv, layer, which, pos0, n, src.data_ptr(), nb, 1, stream))

    def kv_read(self, kv, layer, which, pos0, dst, stream):
        """Cache rows into a device tensor (n_tokens, n_head_kv, head_dim), F32 or F16."""
        kind = _kind(dst)
        _expect(kind is not None, "dst: float32 or float16")
        n, nb = _cache_rows(kv, dst, 4 if kind == MI_TYPE_F32 else 2)
        self.check(self.so.mi_hip_kv_read(kv, layer, which, pos0, n, dst.data_ptr(), kind, nb, stream))

    def kv_keep(self, kv, n_past, idx, stream):
        """Rows n_past + idx[i] become rows n_past + i (idx: whole numbers on the host, increasing)."""
        self.check(self.so.mi_hip_kv_keep(kv, n_past, (ctypes.c_int32 * len(idx))(*idx), len(idx), stream))


_lib = None


def lib():
    global _lib
    if _lib is None:
        _lib = Lib()
    return _lib


_kinds = {}


def _kind(t):
    """The element type of a torch tensor: MI_TYPE_F32, MI_TYPE_F16 or None."""
    if not _kinds:
        import torch
        _kinds.update({torch.float32: MI_TYPE_F32, torch.float16: MI_TYPE_F16})
    return _kinds.get(t.dtype)


def _is_int32(t):
    return t.element_size() == 4 and not t.is_floating_point()


def _expect(ok, what):
    if not ok:
        raise ValueError(what)


def _rows_of(kv, shape):
    # (a handle that is a plain number, or None, does not say its rows' shape)
    rows = getattr(kv, "rows", None)
    return len(shape) == 3 and (rows is None or (shape[1], shape[2]) == rows)


def _cache_rows(kv, t, elt):
    """Tokens and byte strides of a device tensor of rows of the cache."""
    shape = t.shape
    if not _rows_of(kv, shape):
        raise ValueError("rows: shape (n_tokens, n_head_kv, head_dim) of the cache")
    if not t.is_cuda:
        raise ValueError("rows: device memory")
    s2, s1, s0 = t.stride()
    return shape[0], _Strides(s0 * elt, s1 * elt, s2 * elt)


def _expect_one_device(*tensors):
    _expect(len({t.device for t in tensors if t is not None}) <= 1, "tensors of one device")


def nb3_of(t):
    """Byte strides (ne[0] innermost) of a torch tensor shaped (ne2, ne1, ne0)."""
    es = t.element_size()
    s = t.stride()
    return (s[2] * es, s[1] * es, s[0] * es)


def attn_args(q, out, n_rep, n_past, scale, stream, kv=None, layer=0, k=None, v=None, ws=None):
    """Builds AttnArgs from torch tensors q/out shaped (n_tokens, n_head, head_dim) and
    either a cache handle + layer or explicit k/v shaped (n_ctx, n_head_kv, head_dim);
    ws: an optional decode workspace handle (else the cache's, else the library default)."""
    a = AttnArgs()
    a.ws = ws
    if kv is not None:
        a.kv = kv
        a.layer = layer
    else:
        import torch
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.k_nb[:] = nb3_of(k)
        a.v_nb[:] = nb3_of(v)
        a.kv_type = MI_TYPE_F16 if k.dtype == torch.float16 else MI_TYPE_F32
        a.head_dim = k.shape[2]
        a.n_head_kv = k.shape[1]
    a.q = q.data_ptr()
    a.q_nb[:] = nb3_of(q)
    a.out = out.data_ptr()
    a.out_nb[:] = nb3_of(out)
    a.n_tokens, a.n_head = q.shape[0], q.shape[1]
    a.n_rep = n_rep
    a.n_past = n_past
    a.scale = scale
    a.stream = stream
    return a


def rope_args(kv, layer, n_past, n_dims, freq_base, stream, k, v, q=None, q_out=None):
    """Builds RopeArgs from torch tensors shaped (n_tokens, heads, head_dim): k/v
    with the cache's n_head_kv heads, q/q_out (optional) with n_head heads."""
    a = RopeArgs()
    a.kv, a.layer, a.n_past, a.n_dims = kv, layer, n_past, n_dims
    a.freq_base = freq_base
    a.n_tokens = k.shape[0]
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_nb[:] = nb3_of(k)
    a.v_nb[:] = nb3_of(v)
    if q is not None:
        q_out = q if q_out is None else q_out
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
        a.q_nb[:] = nb3_of(q)
        a.q_out_nb[:] = nb3_of(q_out)
        a.n_head = q.shape[1]
    a.stream = stream
    return a


def norm_rope_args(kv, layer, n_past, n_dims, freq_base, stream, k, v, q=None, q_out=None, pos=None, freq=None,
                   q_norm=None, k_norm=None, eps=0.0):
    """Builds NormRopeArgs from torch tensors as rope_args does; pos (n_tokens, int32) and the
    norms' weights (head_dim) are device tensors, freq n_dims / 2 floats on the host."""
    for t in (k, v, q, q_out, q_norm, k_norm):
        _expect(t is None or _kind(t) == MI_TYPE_F32, "q, k, v and the norms' weights: float32")
    _expect(v.shape == k.shape and (q is None or q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2]) and
            (q is None or q_out is None or q_out.shape == q.shape), "q, k, v: shapes of the same tokens and head_dim")
    _expect(all(w is None or (w.numel() == k.shape[2] and w.is_contiguous()) for w in (q_norm, k_norm)),
            "q_norm, k_norm: head_dim weights")
    _expect(_rows_of(kv, k.shape), "k, v: shape (n_tokens, n_head_kv, head_dim) of the cache")
    _expect(pos is None or (_is_int32(pos) and pos.numel() >= k.shape[0] and pos.is_contiguous()),
            "pos: an int32 position for each token")
    _expect_one_device(k, v, q, q_out, pos, q_norm, k_norm)
    _expect(freq is None or len(freq) == n_dims // 2, "freq: n_dims / 2 frequencies")
    a = NormRopeArgs()
    a.kv, a.layer, a.n_past, a.n_dims = kv, layer, n_past, n_dims
    a.freq_base, a.eps = freq_base, eps
    a.n_tokens = k.shape[0]
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_nb[:] = nb3_of(k)
    a.v_nb[:] = nb3_of(v)
    if freq is not None:
        a.freq = (ctypes.c_float * len(freq))(*freq)
    for name, t in (("pos", pos), ("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None:
            setattr(a, name, t.data_ptr())
    if q is not None:
        q_out = q if q_out is None else q_out
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
        a.q_nb[:] = nb3_of(q)
        a.q_out_nb[:] = nb3_of(q_out)
        a.n_head = q.shape[1]
    a.stream = stream
    return a


def tree_masks(bits):
    """An array of TreeMask from one device tensor of 64-bit words (n_tokens, words) per item, or
    None for an item whose tokens are a chain."""
    _expect(all(b is None or (b.element_size() == 8 and not b.is_floating_point() and b.dim() == 2 and b.stride(1) == 1)
                for b in bits), "bits: rows of 64-bit words")
    _expect_one_device(*bits)
    return (TreeMask * len(bits))(*[TreeMask() if b is None else TreeMask(b.data_ptr(), b.stride(0) * 8)
                                    for b in bits])


def logits_args(logits, out, stream, penalties=None, hist=None, hist_off=None, bias_id=None, bias=None,
                bias_off=None, mask=None, ids=None, ws=None):
    """Builds LogitsArgs from device tensors: logits and out (n_rows, n_vocab), penalties
    (n_rows, 3), int32 lists and offsets, mask (n_rows, words) of 32 bits or one row for all."""
    rows, vocab = logits.shape
    _expect(out.shape == logits.shape and all(_kind(t) == MI_TYPE_F32 and (t.stride(1) == 1 or vocab == 1)
                                              for t in (logits, out)), "logits, out: float32 rows (n_rows, n_vocab)")
    for t in (hist, hist_off, bias_id, bias_off, ids):
        _expect(t is None or (_is_int32(t) and t.is_contiguous()), "hist, bias_id, offsets, ids: contiguous int32")
    for t in (penalties, bias):
        _expect(t is None or (_kind(t) == MI_TYPE_F32 and t.is_contiguous()), "penalties, bias: contiguous float32")
    _expect(penalties is None or penalties.numel() == 3 * rows, "penalties: three for each row")
    _expect(all(t is None or t.numel() == rows + 1 for t in (hist_off, bias_off)), "offsets: n_rows + 1")
    _expect(ids is None or ids.numel() >= rows, "ids: one for each row")
    _expect((bias is None) == (bias_id is None) and (bias is None or bias.numel() == bias_id.numel()),
            "bias: a value for each id")
    _expect(mask is None or (_is_int32(mask) and mask.shape[0] in (1, rows) and mask.stride(1) == 1 and
                             mask.shape[1] >= (vocab + 31) // 32), "mask: rows of n_vocab bits in 32-bit words")
    _expect_one_device(logits, out, penalties, hist, hist_off, bias_id, bias, bias_off, mask, ids)
    a = LogitsArgs()
    a.n_rows, a.n_vocab = rows, vocab
    a.logits, a.nb = logits.data_ptr(), logits.stride(0) * 4
    a.out, a.out_nb = out.data_ptr(), out.stride(0) * 4
    for name, t in (("penalties", penalties), ("hist", hist), ("hist_off", hist_off), ("bias_id", bias_id),
                    ("bias", bias), ("bias_off", bias_off), ("mask", mask), ("ids", ids)):
        if t is not None and (t.numel() > 0 or name.endswith("_off")):
            setattr(a, name, t.data_ptr())
    if mask is not None:
        a.mask_nb = mask.stride(0) * 4 if mask.shape[0] > 1 else 0
    if not a.hist:
        a.hist_off = None
    if not a.bias_id:
        a.bias_off = a.bias = None
    a.ws, a.stream = ws, stream
    return a


def _expect_ints(what, *tensors):
    _expect(all(t is None or (_is_int32(t) and t.is_contiguous()) for t in tensors), what + ": contiguous int32")


def _expect_table(table, n_seq):
    _expect(_is_int32(table) and table.dim() == 2 and table.shape[0] == n_seq and
            (table.stride(1) == 1 or table.shape[1] == 1 or n_seq == 0), "table: int32 rows (n_seq, max_pages)")


def page_tables_args(page_size, n_cached, n_new, held, held_out, table, ring, ring_at, ring_at_out, n_kv, q_off, slots,
                     stream, pos=None, seq=None, n_refused=None):
    """Builds PageTablesArgs from int32 device tensors: n_cached, n_new, held, held_out and n_kv (n_seq),
    q_off (n_seq + 1), table (n_seq, max_pages), ring (n_pages), ring_at and ring_at_out (2), slots, pos
    and seq (max_tokens), n_refused (1)."""
    n = n_cached.numel()
    lists = (n_cached, n_new, held, held_out, ring, ring_at, ring_at_out, n_kv, q_off, slots, pos, seq, n_refused)
    _expect_ints("lengths, ring, offsets, slots, pos, seq", *lists)
    _expect(all(t.numel() == n for t in (n_new, held, held_out, n_kv)) and q_off.numel() == n + 1,
            "n_new, held, held_out, n_kv: one for each sequence, q_off one more")
    _expect(ring_at.numel() == 2 and ring_at_out.numel() == 2, "ring_at, ring_at_out: head and tail")
    _expect(all(t is None or t.numel() == slots.numel() for t in (pos, seq)), "pos, seq: one for each slot")
    _expect(n_refused is None or n_refused.numel() >= 1, "n_refused: one number")
    _expect_table(table, n)
    _expect_one_device(table, *lists)
    a = PageTablesArgs()
    a.n_seq, a.page_size, a.n_pages, a.max_pages, a.max_tokens = n, page_size, ring.numel(), table.shape[1], slots.numel()
    for name, t in (("n_cached", n_cached), ("n_new", n_new), ("held", held), ("held_out", held_out), ("table", table),
                    ("ring", ring), ("ring_at", ring_at), ("ring_at_out", ring_at_out), ("n_kv", n_kv), ("q_off", q_off),
                    ("slots", slots), ("pos", pos), ("seq", seq), ("n_refused", n_refused)):
        if t is not None:
            setattr(a, name, t.data_ptr())
    a.table_nb = table.stride(0) * 4
    a.stream = stream
    return a


def paged_append_args(kv, layer, n_dims, freq_base, stream, k, v, slots, pos, q=None, q_out=None, axis=None, freq=None,
                      q_norm=None, k_norm=None, eps=0.0):
    """Builds PagedAppendArgs from torch tensors as norm_rope_args does; slots (n_tokens) and pos (n_axes,
    n_tokens), or (n_tokens,) for one axis, are int32 device tensors, axis n_dims / 2 numbers on the host."""
    n = norm_rope_args(kv, layer, 0, n_dims, freq_base, stream, k, v, q=q, q_out=q_out, freq=freq, q_norm=q_norm,
                       k_norm=k_norm, eps=eps)
    _expect_ints("slots", slots)
    _expect(slots.numel() == n.n_tokens, "slots: a cache row for each token")
    pos = pos if pos.dim() == 2 else pos.reshape(1, -1)
    _expect(_is_int32(pos) and 1 <= pos.shape[0] <= 4 and pos.shape[1] == n.n_tokens and
            (pos.stride(1) == 1 or pos.shape[1] <= 1), "pos: int32 rows (n_axes, n_tokens), up to four")
    _expect_one_device(k, slots, pos)
    _expect(axis is None or len(axis) == n_dims // 2, "axis: one for each of n_dims / 2 pairs")
    a = PagedAppendArgs()
    for name in ("kv", "layer", "n_tokens", "n_dims", "freq_base", "freq", "eps", "q_norm", "k_norm", "n_head", "q", "q_nb",
                 "q_out", "q_out_nb", "k", "k_nb", "v", "v_nb", "stream"):
        setattr(a, name, getattr(n, name))
    a.slots, a.pos = slots.data_ptr(), pos.data_ptr()
    a.n_axes, a.pos_nb = pos.shape[0], pos.stride(0) * 4
    if axis is not None:
        a.axis = (ctypes.c_int32 * len(axis))(*axis)
    return a


def paged_attn_args(kv, layer, q, out, q_off, n_kv, table, scale, stream, max_new=0, ws=None):
    """Builds AttnPagedArgs from device tensors: q and out (n_tokens, n_head, head_dim), int32 q_off
    (n_seq + 1), n_kv (n_seq) and table (n_seq, max_pages)."""
    _expect(all(t.dim() == 3 and _kind(t) == MI_TYPE_F32 for t in (q, out)) and out.shape == q.shape,
            "q, out: float32 (n_tokens, n_head, head_dim)")
    rows = getattr(kv, "rows", None)
    _expect(rows is None or q.shape[2] == rows[1], "q: the cache's head_dim")
    _expect_ints("q_off, n_kv", q_off, n_kv)
    _expect(q_off.numel() == n_kv.numel() + 1, "q_off: one more than n_kv")
    _expect_table(table, n_kv.numel())
    _expect_one_device(q, out, q_off, n_kv, table)
    a = AttnPagedArgs()
    a.kv, a.layer, a.n_seq, a.max_new = kv, layer, n_kv.numel(), max_new
    a.n_tokens, a.n_head = q.shape[0], q.shape[1]
    a.q_off, a.n_kv, a.table = q_off.data_ptr(), n_kv.data_ptr(), table.data_ptr()
    a.table_nb, a.max_pages = table.stride(0) * 4, table.shape[1]
    a.q, a.out = q.data_ptr(), out.data_ptr()
    a.q_nb[:], a.out_nb[:] = nb3_of(q), nb3_of(out)
    a.scale, a.ws, a.stream = scale, ws, stream
    return a


def verify_args(logits, off, token, u, n_path, path, tokens, stream, parent=None, draft=None, temperature=None, ws=None):
    """Builds VerifyArgs from device tensors: logits and draft (n_rows, n_vocab), int32 off (n_seq + 1),
    token and parent (n_rows), n_path (n_seq), path and tokens (n_seq, max_path), float32 u (n_rows) and
    temperature (n_seq)."""
    rows, vocab = logits.shape
    n = n_path.numel()
    _expect(all(t is None or (_kind(t) == MI_TYPE_F32 and t.shape == logits.shape and (t.stride(1) == 1 or vocab == 1))
                for t in (logits, draft)), "logits, draft: float32 rows (n_rows, n_vocab)")
    _expect_ints("off, token, parent, n_path", off, token, parent, n_path)
    _expect(off.numel() == n + 1 and token.numel() == rows and (parent is None or parent.numel() == rows),
            "off: n_seq + 1; token, parent: one for each row")
    for t, m in ((u, rows), (temperature, n)):
        _expect(t is None or (_kind(t) == MI_TYPE_F32 and t.is_contiguous() and t.numel() == m),
                "u, temperature: contiguous float32, one for each row and for each sequence")
    _expect(all(_is_int32(t) and t.dim() == 2 and t.shape[0] == n and (t.stride(1) == 1 or t.shape[1] == 1)
                for t in (path, tokens)) and path.shape == tokens.shape, "path, tokens: int32 rows (n_seq, max_path)")
    _expect_one_device(logits, draft, off, token, parent, u, temperature, n_path, path, tokens)
    a = VerifyArgs()
    a.n_rows, a.n_vocab, a.n_seq, a.max_path = rows, vocab, n, path.shape[1]
    a.logits, a.nb = logits.data_ptr(), logits.stride(0) * 4
    if draft is not None:
        a.draft, a.draft_nb = draft.data_ptr(), draft.stride(0) * 4
    for name, t in (("off", off), ("token", token), ("parent", parent), ("temperature", temperature), ("u", u),
                    ("n_path", n_path), ("path", path), ("tokens", tokens)):
        if t is not None:
            setattr(a, name, t.data_ptr())
    a.path_nb, a.tokens_nb = path.stride(0) * 4, tokens.stride(0) * 4
    a.ws, a.stream = ws, stream
    return a


def make_tensor(data_ptr, ne, nb, type_=MI_TYPE_F32, op=MI_OP_NONE, src=(), params=()):
    """An mi_tensor descriptor (ne/nb in engine order, ne[0] innermost)."""
    t = MiTensor()
    t.type = type_
    ne = list(ne) + [1] * (4 - len(ne))
    nb = list(nb)
    while len(nb) < 4:
        nb.append(nb[-1] * ne[len(nb) - 1])
    t.ne[:] = ne
    t.nb[:] = nb
    t.op = op
    t.data = data_ptr
    for i, s in enumerate(src):
        t.src[i] = ctypes.pointer(s)
    for i, p in enumerate(params):
        if isinstance(p, float):
            t.op_params[i] = ctypes.c_int32.from_buffer(ctypes.c_float(p)).value
        else:
            t.op_params[i] = p
    return t
