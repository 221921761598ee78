"""ctypes binding of libq4gpu (include/q4_gpu.h) plus a thin host-side mirror of the reference
engine's session KV interface (src/q4_fwd.c: kv_write / kv_at / qsa_attend / q4_sess_save).

Device memory, streams and process groups come from PyTorch; every byte of arithmetic on the
path is done by the CUDA library.  There is no fallback: if the shared library is missing or no
CUDA device is present, loading / init raises.
"""
import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "lib", "libq4gpu.so")
HEADER_PATH = os.path.join(os.path.dirname(os.path.dirname(_HERE)), "include", "q4_gpu.h")

KIND_F32, KIND_F16, KIND_Q8 = 0, 1, 2
KIND_NAMES = {"f32": 0, "fp32": 0, "f16": 1, "fp16": 1, "q8": 2, "q8_0": 2}

_b, _v, _u32, _i32, _u64, _f, _sz, _i, _d = (C.c_bool, C.c_void_p, C.c_uint32, C.c_int32, C.c_uint64,
                                            C.c_float, C.c_size_t, C.c_int, C.c_double)

# name -> (restype, argtypes); mirrors include/q4_gpu.h declaration by declaration
SIGNATURES = {
    "q4_hip_init": (_b, []), "q4_hip_shutdown": (None, []), "q4_hip_ok": (_b, []),
    "q4_hip_malloc": (_v, [_sz]), "q4_hip_free": (None, [_v]),
    "q4_hip_h2d": (_b, [_v, _v, _sz]), "q4_hip_d2h": (_b, [_v, _v, _sz]),
    "q4_hip_d2h_async": (_b, [_v, _v, _u64]), "q4_hip_h2d_async": (_b, [_v, _v, _u64]),
    "q4_hip_stream_sync": (_b, []),
    "q4_hip_copy_h2d": (_b, [_v, _v, _sz]), "q4_hip_copy_wait": (None, []), "q4_gpu_copy_stream": (_v, []),
    "q4_gpu_copy_d2h": (_b, [_v, _v, _sz]), "q4_gpu_download_stream": (_v, []),
    "q4_gpu_graph_apart": (_u32, []), "q4_gpu_graph_ahead": (_u32, []), "q4_gpu_prefill_layout": (None, [_v, _v, _v]),
    "q4_gpu_pipe_create": (_v, []), "q4_gpu_pipe_destroy": (None, [_v]),
    "q4_gpu_pipe_upload": (_b, [_v, _v, _v, _sz]), "q4_gpu_pipe_run": (_b, [_v, _v, _v, _v, _sz]),
    "q4_gpu_pipe_sync": (_b, [_v]),
    "q4_hip_copy": (_b, [_v, _v, _u64]), "q4_hip_fill": (_b, [_v, _f, _u64]),
    "q4_hip_sync": (None, []), "q4_hip_clear": (None, []),
    "q4_hip_pos_push": (None, [_i32]), "q4_hip_capturing": (_i, []), "q4_hip_pos_dev_ok": (_i, []),
    "q4_hip_graph_begin": (_i, []), "q4_hip_graph_end": (_v, []), "q4_hip_graph_nodes": (_u32, [_v]),
    "q4_hip_graph_launch": (_b, [_v]), "q4_hip_graph_free": (None, [_v]),
    "q4_hip_f32_to_f16": (_b, [_v, _v, _u64]), "q4_hip_f32_to_q8": (_b, [_v, _v, _u64]),
    "q4_hip_f32_to_f16_d": (_b, [_v, _u32, _v, _u64]),
    "q4_hip_kv_append_d": (_b, [_v, _v, _v, _v, _u32, _u32, _i]),
    "q4_hip_qsa_q_prep": (_b, [_v, _v, _v, _v, _u32, _u32, _u32, _i32, _f, _f]),
    "q4_hip_qsa_q_prep_n": (_b, [_v, _v, _v, _v, _u32, _u32, _u32, _i32, _f, _f, _u32]),
    "q4_hip_qsa_q_prep_d": (_b, [_v, _v, _v, _v, _u32, _u32, _u32, _f, _f]),
    "q4_hip_qsa_k_prep": (_b, [_v, _v, _u32, _u32, _u32, _i32, _f, _f]),
    "q4_hip_qsa_k_prep_n": (_b, [_v, _v, _u32, _u32, _u32, _i32, _f, _f, _u32]),
    "q4_hip_qsa_k_prep_d": (_b, [_v, _v, _u32, _u32, _u32, _f, _f]),
    "q4_hip_qsa_decode": (_b, [_v, _v, _v, _v, _v, _u32, _u32, _u32, _u32, _u32, _f, _i]),
    "q4_hip_qsa_decode_n": (_b, [_v, _v, _v, _v, _v, _u32, _u32, _u32, _u32, _u32, _u32, _f, _i]),
    "q4_hip_qsa_decode_idx": (_b, [_v, _v, _v, _v, _v, _v, _u32, _u32, _u32, _u32, _u32, _u32, _f, _i]),
    "q4_hip_qsa_topk_alloc": (_b, []),
    "q4_gpu_last_error": (_u32, []), "q4_gpu_stream": (_v, []), "q4_gpu_set_stream": (_b, [_v]),
    "q4_gpu_device": (_i, []), "q4_gpu_pos_word": (_v, []),
    "q4_gpu_kv_bytes": (_u64, [_u32, _u32, _u32, _u32, _i]),
    "q4_gpu_kv_create": (_v, [_u32, _u32, _u32, _u32, _i]), "q4_gpu_kv_destroy": (None, [_v]),
    "q4_gpu_kv_append": (_b, [_v, _u32, _v, _v, _u32, _u32]),
    "q4_gpu_kv_append_d": (_b, [_v, _u32, _v, _v]),
    "q4_gpu_kv_prep_append": (_b, [_v, _u32, _v, _v, _v, _u32, _f, _f, _u32, _u32]),
    "q4_gpu_kv_prep_append_d": (_b, [_v, _u32, _v, _v, _v, _u32, _f, _f]),
    "q4_gpu_kv_export": (_b, [_v, _u32, _i, _u32, _u32, _v]),
    "q4_gpu_kv_import": (_b, [_v, _u32, _i, _u32, _u32, _v]),
    "q4_gpu_kv_snapshot_bytes": (_u64, [_v, _u32]),
    "q4_gpu_kv_save": (_b, [_v, _u32, _v, _i]), "q4_gpu_kv_restore": (_b, [_v, _u32, _v, _i]),
    "q4_gpu_kv_write_fd": (_b, [_v, _u32, _i]), "q4_gpu_kv_read_fd": (_b, [_v, _u32, _i]),
    "q4_gpu_sess_file_bytes": (_u64, [_v, _u32, _v]),
    "q4_gpu_sess_file_write": (_b, [_v, _u32, _v, C.c_char_p]),
    "q4_gpu_sess_file_read": (_i, [_v, _v, _v, _i, C.c_char_p]),
    "q4_gpu_sess_file_peek_ids": (_i, [_v, C.c_char_p, _v, _i, _v, _v, _v]),
    "q4_gpu_kv_decode": (_b, [_v, _u32, _v, _i, _v, _v, _u32, _v, _u32, _u32, _u32, _f]),
    "q4_gpu_kv_decode_noalloc": (_b, [_v, _u32, _v, _i, _v, _v, _u32, _v, _u32, _u32, _u32, _f]),
    "q4_gpu_kv_decode_idx_n": (_b, [_v, _u32, _v, _i, _v, _v, _u32, _v, _u32, _u32, _u32, _u32, _f]),
    "q4_gpu_kv_decode_partial": (_b, [_v, _u32, _v, _i, _v, _u32, _v, _u32, _u32, _u32, _f]),
    "q4_gpu_lse_merge": (_b, [_v, _u32, _u32, _u32, _v, _v]),
    "q4_hip_qsa_pool": (_b, [_v, _v, _v, _u32, _u32, _u32, _u32, _u32, _f, _f]),
    "q4_hip_qsa_pool_d": (_b, [_v, _v, _v, _u32, _u32, _u32, _f, _f]),
    "q4_hip_qsa_score": (_b, [_v, _v, _v, _u32, _u32, _u32, _u32, _u32, _u32, _u32]),
    "q4_hip_qsa_score_d": (_b, [_v, _v, _v, _u32, _u32, _u32, _u32]),
    "q4_hip_qsa_topk": (_b, [_v, _v, _u32, _u32, _u32, _u32, _u32, _u32, _u32]),
    "q4_hip_qsa_topk_d": (_b, [_v, _v, _u32, _u32, _u32, _u32]),
    "q4_gpu_qsa_select_batch": (_b, [_v, _v, _v, _v, _v, _u32, _u32, _u32, _u32, _u32, _u32, _u32]),
    "q4_gpu_xchg_create": (_v, [_u32, _u32, _u32, _u32, _u32]), "q4_gpu_xchg_destroy": (None, [_v]),
    "q4_gpu_xchg_handle": (_b, [_v, _v]), "q4_gpu_xchg_window": (_v, [_v]),
    "q4_gpu_xchg_attach": (_b, [_v, _u32, _v]), "q4_gpu_xchg_attach_ptr": (_b, [_v, _u32, _v]),
    "q4_gpu_xchg_set_timeout_ms": (_b, [_v, _u32]),
    "q4_gpu_kv_decode_xchg": (_b, [_v, _v, _u32, _v, _i, _v, _v, _u32, _f, _i]),
    "q4_gpu_comm_unique_id": (_b, [_v]), "q4_gpu_comm_create": (_v, [_v, _u32, _u32]),
    "q4_gpu_comm_destroy": (None, [_v]), "q4_gpu_comm_allgather_merge": (_b, [_v, _v, _v, _u32, _u32, _v, _v]),
    "q4_gpu_kv_prefill": (_b, [_v, _u32, _v, _v, _v, _u32, _u32, _u32, _f]),
    "q4_gpu_batch_create": (_v, [_u32]), "q4_gpu_batch_destroy": (None, [_v]),
    "q4_gpu_batch_bind": (_b, [_v, _u32, _v]), "q4_gpu_batch_set_pos": (_b, [_v, _v, _u32]),
    "q4_gpu_batch_advance": (_b, [_v, _i32]),
    "q4_gpu_batch_append": (_b, [_v, _u32, _v, _v]),
    "q4_gpu_batch_decode": (_b, [_v, _u32, _v, _i, _v, _v, _v, _u32, _u32, _u32, _u32, _f]),
    "q4_gpu_batch_append_decode": (_b, [_v, _u32, _v, _v, _v, _i, _v, _v, _v, _u32, _u32, _u32, _u32, _f]),
    "q4_gpu_kv_append_decode_d": (_b, [_v, _u32, _v, _v, _v, _i, _v, _v, _u32, _v, _u32, _u32, _f]),
    "q4_gpu_pages_bytes": (_u64, [_u32, _u32, _u32, _u32, _u32, _i]),
    "q4_gpu_pages_plan": (_b, [_v, _v, _v, _u32, _v, _u32, _v, _v, _v, _v, _u32]),
    "q4_gpu_pages_trim": (_b, [_v, _v, _v, _u32, _v, _u32]),
    "q4_gpu_pages_append": (_b, [_v, _u32, _v, _v, _v, _u32]),
    "q4_gpu_pages_gather": (_b, [_v, _u32, _v, _u32, _v, _v]),
    "q4_gpu_pages_attend": (_b, [_v, _u32, _v, _i, _v, _v, _i, _u32, _v, _v, _u32, _u32, _v, _u32, _u32, _f]),
    "q4_gpu_rope_set": (_b, [_v, _u32, _i, _d, _i, _d, _d, _d, _d, _d]),
    "q4_gpu_pages_prep": (_b, [_v, _u32, _v, _v, _v, _i, _u64, _u64, _u32, _v, _v, _f, _v, _v, _v, _u32, _v, _i, _v]),
    "q4_gpu_pages_fork": (_b, [_v, _v, _v, _u32, _v, _v, _v, _u32, _v, _u32]),
    "q4_gpu_pages_release": (_b, [_v, _v, _v, _v, _u32, _v, _u32]),
    "q4_gpu_pages_compact": (_b, [_v, _v, _v, _u32, _v, _u32, _v]),
    "q4_gpu_verify": (_b, [_v, _i, _u64, _v, _u64, _u32, _v, _v, _u32, _u32, _v, _v, _v, _v, _v, _v, _v, _v]),
}


class PagesDesc(C.Structure):
    """q4_gpu_pages of include/q4_gpu.h: a pool of pages in the caller's memory"""
    _fields_ = [("mem", C.c_void_p), ("free_list", C.c_void_p), ("n_free", C.c_void_p), ("n_layers", C.c_uint32), ("n_kvh", C.c_uint32),
                ("hd", C.c_uint32), ("n_pages", C.c_uint32), ("page_rows", C.c_uint32), ("kind", C.c_int)]


class Rope(C.Structure):
    """q4_gpu_rope of include/q4_gpu.h: how positions turn the first n_rot dims of a head, in pairs (2 i, 2 i + 1) or, half, (i, i + n_rot / 2).
    scaling: None, or for contexts longer than orig positions by factor "linear", "ramp" (over the pairs between those that turn fast and slow
    times in orig positions) or "smooth" (over the turns from slow to fast).  Needs no device."""
    _fields_ = [("n_rot", C.c_uint32), ("half", C.c_int32), ("mag", C.c_float), ("reserved", C.c_uint32), ("turn", C.c_uint64 * 128)]
    SCALINGS = {None: 0, "linear": 1, "ramp": 2, "smooth": 3}

    def __init__(self, n_rot, base, half=False, scaling=None, factor=1.0, orig=0.0, fast=32.0, slow=1.0, mag=1.0):
        super().__init__()
        if scaling not in self.SCALINGS or not 0 <= n_rot <= 256:
            raise RuntimeError("a scaling of %s and up to 256 dims are needed, not %r and %r" % (list(self.SCALINGS), scaling, n_rot))
        self.p = C.addressof(self)
        check(load().q4_gpu_rope_set(self.p, n_rot, int(half), base, self.SCALINGS[scaling], factor, orig, fast, slow, mag), "q4_gpu_rope_set")


class SessDesc(C.Structure):
    """q4_gpu_sess_desc of include/q4_gpu.h: the host's part of a version-5 session file"""
    _fields_ = [("bytes_total", C.c_uint64), ("n_layer", C.c_uint32), ("n_expert", C.c_uint32), ("pos", C.c_uint32),
                ("n_gdn", C.c_uint32), ("n_v_h", C.c_uint32), ("d_v", C.c_uint32), ("conv_hist", C.c_uint32),
                ("conv_ch", C.c_uint32), ("hc_dim", C.c_uint32), ("prompt_n", C.c_uint32), ("nmsg", C.c_uint32),
                ("user_hash", C.c_uint64), ("ids", C.c_void_p), ("n_ids", C.c_uint32), ("ple_hist", C.c_int32 * 8),
                ("state_a", C.c_void_p), ("state_a_bytes", C.c_uint64), ("state_b", C.c_void_p),
                ("state_b_bytes", C.c_uint64), ("idx_dim", C.c_uint32), ("idx_has_raw", C.c_uint32),
                ("idx_raw", C.c_void_p), ("idx_raw_bytes", C.c_uint64)]


_lib = None


def load():
    """dlopen libq4gpu.so and type every entry point.  Raises if the library was not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("libq4gpu.so is not built (%s): run __graft_entry__.build() or "
                               "`make -C suzuqu-engine-4exp_b200/csrc`; there is no fallback path" % LIB_PATH)
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def init():
    """q4_hip_init(); raises when no sm_100 device is usable."""
    L = load()
    if not L.q4_hip_init():
        raise RuntimeError("q4_hip_init failed: no usable CUDA device (libq4gpu has no CPU path)")
    return L


def _ptr(t):
    """Device (or host) address of a torch tensor / numpy array / int / None."""
    if t is None or isinstance(t, int):
        return t
    try:
        return t.data_ptr()
    except AttributeError:
        return t.ctypes.data


def _dense(t, dtype, n, gpu):
    """address of a dense tensor of that type, of n numbers or more, on that GPU; None stays None"""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() < n or t.get_device() != gpu or not t.is_contiguous():
        raise RuntimeError("a dense tensor of %s on GPU %d with %d numbers is needed, not one of %s on %s, %s with strides %s"
                           % (dtype, gpu, n, t.dtype, t.device, tuple(t.shape), t.stride()))
    return t.data_ptr()


def _rows(t, dtype, n_rows, width, gpu):
    """address and row stride of a tensor [n_rows or more][width or more] of that type on that GPU, whose rows are dense"""
    if t.dim() == 2:
        (n, w), (apart, one) = t.shape, t.stride()
        if n <= 1:                                                         # a single row has no stride
            apart = width
        if t.dtype is dtype and t.get_device() == gpu and n >= n_rows and w >= width and (one == 1 or w <= 1) and apart >= width:
            return t.data_ptr(), apart
    raise RuntimeError("rows of %d numbers of %s on GPU %d are needed, %d of them, not one of %s on %s, %s with strides %s"
                       % (width, dtype, gpu, n_rows, t.dtype, t.device, tuple(t.shape), t.stride()))


def check(ok, what):
    if not ok:
        raise RuntimeError("%s failed (status %#x)" % (what, load().q4_gpu_last_error()))


def use_torch_stream():
    """Run the library on torch's current CUDA stream so torch ops and library calls are ordered."""
    import torch
    # torch's default stream has handle 0; its explicit CUDA name is cudaStreamLegacy (0x1)
    check(load().q4_gpu_set_stream(torch.cuda.current_stream().cuda_stream or 1), "q4_gpu_set_stream")


class KVStore:
    """One session's KV cache in the library's planar layout -- the role of q4_sess's
    d_qsa_k / d_qsa_v / kv_kind / kv_bpt / max_kv fields (src/q4_fwd.c:26-57,1944-1950)."""

    def __init__(self, n_layers, n_kvh, hd, max_kv, kind=KIND_Q8):
        self.L = init()
        self.n_layers, self.n_kvh, self.hd, self.max_kv, self.kind = n_layers, n_kvh, hd, max_kv, kind
        self.h = self.L.q4_gpu_kv_create(n_layers, n_kvh, hd, max_kv, kind)
        if not self.h:
            raise RuntimeError("q4_gpu_kv_create failed (status %#x)" % self.L.q4_gpu_last_error())
        self.n_kv = 0

    def close(self):
        if self.h:
            self.L.q4_gpu_kv_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def token_bytes(self):
        """kv_token_bytes (src/q4_fwd.c:644-650): bytes per token per cache in the reference layout."""
        kvw = self.n_kvh * self.hd
        return kvw // 32 * 34 if self.kind == KIND_Q8 else kvw * (2 if self.kind == KIND_F16 else 4)

    def bytes(self):
        return self.L.q4_gpu_kv_bytes(self.n_layers, self.n_kvh, self.hd, self.max_kv, self.kind)

    def append(self, layer, k, v, pos0, n_tok):
        check(self.L.q4_gpu_kv_append(self.h, layer, _ptr(k), _ptr(v), pos0, n_tok), "q4_gpu_kv_append")

    def append_d(self, layer, k, v):
        check(self.L.q4_gpu_kv_append_d(self.h, layer, _ptr(k), _ptr(v)), "q4_gpu_kv_append_d")

    def export(self, layer, which, tok0, n_tok, dst):
        check(self.L.q4_gpu_kv_export(self.h, layer, which, tok0, n_tok, _ptr(dst)), "q4_gpu_kv_export")

    def import_(self, layer, which, tok0, n_tok, src):
        check(self.L.q4_gpu_kv_import(self.h, layer, which, tok0, n_tok, _ptr(src)), "q4_gpu_kv_import")

    def snapshot_bytes(self, n_kv):
        return self.L.q4_gpu_kv_snapshot_bytes(self.h, n_kv)

    def save(self, n_kv, buf, host=False):
        check(self.L.q4_gpu_kv_save(self.h, n_kv, _ptr(buf), int(host)), "q4_gpu_kv_save")

    def restore(self, n_kv, buf, host=False):
        check(self.L.q4_gpu_kv_restore(self.h, n_kv, _ptr(buf), int(host)), "q4_gpu_kv_restore")

    def write_fd(self, n_kv, fd):
        check(self.L.q4_gpu_kv_write_fd(self.h, n_kv, fd), "q4_gpu_kv_write_fd")

    def read_fd(self, n_kv, fd):
        check(self.L.q4_gpu_kv_read_fd(self.h, n_kv, fd), "q4_gpu_kv_read_fd")

    def sess_file_write(self, n_kv, desc, path):
        """the whole version-5 session file (q4_sess_save); desc: SessDesc"""
        check(self.L.q4_gpu_sess_file_write(self.h, n_kv, C.byref(desc), os.fsencode(path)), "q4_gpu_sess_file_write")

    def sess_file_read(self, desc, ids, path):
        """q4_sess_restore: the saved prefix length, or 0 when the file is refused; ids: int32 numpy array"""
        return self.L.q4_gpu_sess_file_read(self.h, C.byref(desc), ids.ctypes.data, len(ids), os.fsencode(path))

    def decode(self, layer, q, out, n_head, scale, gate=None, idx=None, width=0, idx_kvh_stride=0,
               n_kv=0, q_bf16=False):
        check(self.L.q4_gpu_kv_decode(self.h, layer, _ptr(q), int(q_bf16), _ptr(gate), _ptr(out), n_head,
                                      _ptr(idx), width, idx_kvh_stride, n_kv, scale), "q4_gpu_kv_decode")

    def prefill(self, layer, q_bf16, out_bf16, n_head, n_tok, kv_base, scale, gate=None):
        """causal attention of n_tok queries (bf16) over rows [0, kv_base + t + 1); bf16 output"""
        check(self.L.q4_gpu_kv_prefill(self.h, layer, _ptr(q_bf16), _ptr(gate), _ptr(out_bf16), n_head, n_tok,
                                       kv_base, scale), "q4_gpu_kv_prefill")

    def append_decode_d(self, layer, k, v, q, out, n_head, scale, gate=None, idx=None, width=0, idx_kvh_stride=0,
                        q_bf16=False):
        """append at the device position word + decode over rows [0, position] in one call"""
        check(self.L.q4_gpu_kv_append_decode_d(self.h, layer, _ptr(k), _ptr(v), _ptr(q), int(q_bf16), _ptr(gate),
                                               _ptr(out), n_head, _ptr(idx), width, idx_kvh_stride, scale),
              "q4_gpu_kv_append_decode_d")

    def decode_idx_n(self, layer, q, out, n_head, scale, idx, width, n_tok, idx_tok_stride, idx_kvh_stride=0,
                     gate=None, q_bf16=False):
        """sparse prefill: n_tok queries, each over the rows of its own list (one launch)"""
        check(self.L.q4_gpu_kv_decode_idx_n(self.h, layer, _ptr(q), int(q_bf16), _ptr(gate), _ptr(out), n_head,
                                            _ptr(idx), width, idx_kvh_stride, idx_tok_stride, n_tok, scale),
              "q4_gpu_kv_decode_idx_n")

    def decode_partial(self, layer, q, part, n_head, scale, idx=None, width=0, idx_kvh_stride=0, n_kv=0,
                       q_bf16=False):
        check(self.L.q4_gpu_kv_decode_partial(self.h, layer, _ptr(q), int(q_bf16), _ptr(part), n_head,
                                              _ptr(idx), width, idx_kvh_stride, n_kv, scale),
              "q4_gpu_kv_decode_partial")


class Exchange:
    """Exchange window of one rank of a sequence-sharded decode (q4_gpu_xchg_*): the decode kernel
    pushes its record into the peers' windows and merges theirs, one launch per layer."""
    FUSED, PUSH, MERGE = 0, 1, 2

    def __init__(self, rank, world, n_head, n_kvh, hd):
        self.L = init()
        self.rank, self.world = rank, world
        self.h = self.L.q4_gpu_xchg_create(rank, world, n_head, n_kvh, hd)
        if not self.h:
            raise RuntimeError("q4_gpu_xchg_create failed (status %#x)" % self.L.q4_gpu_last_error())

    def handle(self):
        """the 64-byte IPC handle of the local window"""
        buf = C.create_string_buffer(64)
        check(self.L.q4_gpu_xchg_handle(self.h, C.cast(buf, C.c_void_p)), "q4_gpu_xchg_handle")
        return bytes(buf.raw)

    def window(self):
        return self.L.q4_gpu_xchg_window(self.h)

    def attach(self, peer_rank, handle):
        buf = C.create_string_buffer(bytes(handle), 64)
        check(self.L.q4_gpu_xchg_attach(self.h, peer_rank, C.cast(buf, C.c_void_p)), "q4_gpu_xchg_attach")

    def attach_ptr(self, peer_rank, window):
        check(self.L.q4_gpu_xchg_attach_ptr(self.h, peer_rank, window), "q4_gpu_xchg_attach_ptr")

    def attach_all(self, dist):
        """exchange the handles over a torch.distributed process group (host side, once) and open them"""
        handles = [None] * self.world
        dist.all_gather_object(handles, self.handle())
        for r, hd_ in enumerate(handles):
            if r != self.rank:
                self.attach(r, hd_)
        dist.barrier()

    def set_timeout_ms(self, ms):
        check(self.L.q4_gpu_xchg_set_timeout_ms(self.h, ms), "q4_gpu_xchg_set_timeout_ms")

    def decode(self, store, layer, q, out, scale, n_kv, gate=None, q_bf16=False, phase=0):
        check(self.L.q4_gpu_kv_decode_xchg(store.h if store is not None else None, self.h, layer, _ptr(q),
                                           int(q_bf16), _ptr(gate), _ptr(out), n_kv, scale, phase),
              "q4_gpu_kv_decode_xchg")

    def close(self):
        if self.h:
            self.L.q4_gpu_xchg_destroy(self.h)
            self.h = None


class Comm:
    """NCCL communicator of the library (q4_gpu_comm_*), built from a unique id that the host distributes --
    here over a torch.distributed process group, by broadcast from rank 0."""

    def __init__(self, rank, world, dist=None):
        self.L = init()
        buf = C.create_string_buffer(128)
        if rank == 0:
            check(self.L.q4_gpu_comm_unique_id(C.cast(buf, C.c_void_p)), "q4_gpu_comm_unique_id")
        box = [bytes(buf.raw)]
        if world > 1:
            dist.broadcast_object_list(box, src=0)
        idbuf = C.create_string_buffer(box[0], 128)
        self.h = self.L.q4_gpu_comm_create(C.cast(idbuf, C.c_void_p), rank, world)
        if not self.h:
            raise RuntimeError("q4_gpu_comm_create failed (status %#x)" % self.L.q4_gpu_last_error())
        self.world = world

    def allgather_merge(self, part, parts_all, n_head, hd, out, gate=None):
        check(self.L.q4_gpu_comm_allgather_merge(self.h, _ptr(part), _ptr(parts_all), n_head, hd, _ptr(gate), _ptr(out)),
              "q4_gpu_comm_allgather_merge")

    def close(self):
        if self.h:
            self.L.q4_gpu_comm_destroy(self.h)
            self.h = None


class Batch:
    """Concurrent sessions decoded with one launch per layer."""

    def __init__(self, stores):
        self.L = init()
        self.stores = list(stores)
        self.h = self.L.q4_gpu_batch_create(len(self.stores))
        if not self.h:
            raise RuntimeError("q4_gpu_batch_create failed")
        for i, s in enumerate(self.stores):
            check(self.L.q4_gpu_batch_bind(self.h, i, s.h), "q4_gpu_batch_bind")

    def close(self):
        if self.h:
            self.L.q4_gpu_batch_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_pos(self, pos):
        arr = (C.c_int32 * len(pos))(*[int(p) for p in pos])
        check(self.L.q4_gpu_batch_set_pos(self.h, arr, len(pos)), "q4_gpu_batch_set_pos")

    def advance(self, delta=1):
        """pos[s] += delta on the device (capturable)"""
        check(self.L.q4_gpu_batch_advance(self.h, delta), "q4_gpu_batch_advance")

    def append(self, layer, k, v):
        check(self.L.q4_gpu_batch_append(self.h, layer, _ptr(k), _ptr(v)), "q4_gpu_batch_append")

    def decode(self, layer, q, out, n_head, scale, gate=None, idx=None, width=0, idx_kvh_stride=0,
               idx_sess_stride=0, q_bf16=False):
        check(self.L.q4_gpu_batch_decode(self.h, layer, _ptr(q), int(q_bf16), _ptr(gate), _ptr(out), _ptr(idx),
                                         width, idx_kvh_stride, idx_sess_stride, n_head, scale),
              "q4_gpu_batch_decode")

    def append_decode(self, layer, k, v, q, out, n_head, scale, gate=None, idx=None, width=0, idx_kvh_stride=0,
                      idx_sess_stride=0, q_bf16=False):
        """append + decode in one call (one launch per layer at hd 128 and 256)"""
        check(self.L.q4_gpu_batch_append_decode(self.h, layer, _ptr(k), _ptr(v), _ptr(q), int(q_bf16), _ptr(gate),
                                                _ptr(out), _ptr(idx), width, idx_kvh_stride, idx_sess_stride,
                                                n_head, scale), "q4_gpu_batch_append_decode")


class PagePool:
    """A paged KV cache for many requests (q4_gpu_pages_*).  Arrays are dense torch tensors on the library's GPU, others are refused
    (RuntimeError), as are ones too small for the call; the pool's memory and its stack of free pages are allocated here unless they
    are given.  Per step: plan, then append and attend for every layer."""

    def __init__(self, n_layers, n_kvh, hd, n_pages, page_rows=64, kind=KIND_Q8, mem=None, free=None, n_free=None, shares=None):
        import torch
        self.L = init()
        size = self.L.q4_gpu_pages_bytes(n_layers, n_kvh, hd, n_pages, page_rows, kind)
        if not size:
            raise RuntimeError("q4_gpu_pages_bytes: a pool of kind f16 or q8_0, hd 64 / 128 / 256, page_rows 16 .. 256 is needed")
        self.gpu = gpu = self.L.q4_gpu_device()
        on = torch.device("cuda", gpu)
        own_mem = free is None and mem is None and n_free is None
        if own_mem:
            mem = torch.empty(size, dtype=torch.uint8, device=on)
            free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=on)   # page 0 is on top
            n_free = torch.full((1,), n_pages, dtype=torch.int32, device=on)
            shares = torch.zeros(3 * n_pages, dtype=torch.int32, device=on) if shares is None else shares
        if (free is None) != (n_free is None):
            raise RuntimeError("the stack of free pages and its height go together")
        if mem is not None and mem.numel() * mem.element_size() < size:
            raise RuntimeError("the pool's memory is smaller than q4_gpu_pages_bytes (%d)" % size)
        self.mem, self.free, self.n_free, self.shares = mem, free, n_free, shares   # shares: holders besides the first, fork and release count them
        self.n_layers, self.n_kvh, self.hd, self.n_pages, self.page_rows, self.kind = n_layers, n_kvh, hd, n_pages, page_rows, kind
        at = (_dense(mem, None if mem is None else mem.dtype, 1, gpu), _dense(free, torch.int32, n_pages, gpu), _dense(n_free, torch.int32, 1, gpu))
        self.desc = PagesDesc(*at, n_layers, n_kvh, hd, n_pages, page_rows, kind)
        self.p, self.width, self.shared = C.addressof(self.desc), n_kvh * hd, _dense(shares, torch.int32, 3 * n_pages, gpu)
        self.calls = [getattr(self.L, "q4_gpu_pages_" + name) for name in ("plan", "trim", "append", "gather", "attend", "prep", "fork", "release", "compact")]
        self.i32, self.f32, self.bf16 = torch.int32, torch.float32, torch.bfloat16

    # a call costs the host as much as a small launch the device: addresses are taken once, functions looked up above

    def plan(self, rows, add, table, start, slot, pos, req):
        """pages for add[r] more tokens of every request, and the step's maps; table [n_req][stride], slot / pos / req [max_tok].  Request r
        then holds start[r + 1] - start[r] rows more: all of add[r], or none where pages or max_tok ran out"""
        i, gpu, (n, stride), m = self.i32, self.gpu, table.shape, slot.shape[0]
        if not self.calls[0](self.p, _dense(rows, i, n, gpu), _dense(add, i, n, gpu), n, _dense(table, i, n * stride, gpu), stride, _dense(start, i, n + 1, gpu),
                             _dense(slot, i, m, gpu), _dense(pos, i, m, gpu), _dense(req, i, m, gpu), m):
            check(False, "q4_gpu_pages_plan")

    def trim(self, rows, keep, table):
        """the pages behind the first keep[r] of rows[r] rows go back"""
        i, gpu, (n, stride) = self.i32, self.gpu, table.shape
        if not self.calls[1](self.p, _dense(rows, i, n, gpu), _dense(keep, i, n, gpu), n, _dense(table, i, n * stride, gpu), stride):
            check(False, "q4_gpu_pages_trim")

    def append(self, layer, k, v, slot):
        """k, v [slot.shape[0]][n_kvh * hd] fp32; slots below 0 are skipped"""
        gpu, m = self.gpu, slot.shape[0]
        x = m * self.width
        if not self.calls[2](self.p, layer, _dense(k, self.f32, x, gpu), _dense(v, self.f32, x, gpu), _dense(slot, self.i32, m, gpu), m):
            check(False, "q4_gpu_pages_append")

    def gather(self, layer, slot, k, v):
        """the rows of the slots as fp32, the reverse of append; k or v may be None"""
        gpu, m = self.gpu, slot.shape[0]
        x = m * self.width
        if not self.calls[3](self.p, layer, _dense(slot, self.i32, m, gpu), m, _dense(k, self.f32, x, gpu), _dense(v, self.f32, x, gpu)):
            check(False, "q4_gpu_pages_gather")

    def attend(self, layer, q, out, rows, start, table, n_head, scale, gate=None, max_add=0):
        """attention of the step's tokens: q, out [n_tok][n_head][hd], bf16 or fp32; rows as they were given to plan"""
        i, gpu, (n, stride), x, per = self.i32, self.gpu, table.shape, q.numel(), n_head * self.hd
        if per <= 0 or x % per:
            raise RuntimeError("queries of %s are no tokens of %d heads of %d" % (tuple(q.shape), n_head, self.hd))
        q_bf16, out_bf16 = q.dtype is self.bf16, out.dtype is self.bf16
        if not self.calls[4](self.p, layer, _dense(q, self.bf16 if q_bf16 else self.f32, x, gpu), q_bf16, _dense(gate, self.f32, x, gpu),
                             _dense(out, self.bf16 if out_bf16 else self.f32, x, gpu), out_bf16, n_head, _dense(rows, i, n, gpu), _dense(start, i, n + 1, gpu), n, x // per,
                             _dense(table, i, n * stride, gpu), stride, max_add, scale):
            check(False, "q4_gpu_pages_attend")

    def prep(self, layer, q, k, v, q_out, pos, slot, rope, wq=None, wk=None, eps=1e-6, gate=None):
        """the projections' rows made ready for attend: q [n_tok][n_head * hd], or [n_head][q | gate] where gate is given, k and v [n_tok][n_kvh * hd], fp32 or
        bf16, each dense in its rows (k and v at one stride); q_out [n_tok][n_head][hd], gate likewise fp32; pos and slot as plan made them; wq, wk [hd]; eps None: no norm"""
        gpu, m, dtype = self.gpu, pos.shape[0], q.dtype
        if q_out.dim() != 3 or q_out.shape[2] != self.hd or (dtype is not self.f32 and dtype is not self.bf16):
            raise RuntimeError("queries of %s are no heads of %d, or those of %s neither fp32 nor bf16" % (tuple(q_out.shape), self.hd, dtype))
        n_head, q_bf16 = q_out.shape[1], q_out.dtype is self.bf16
        x = n_head * self.hd
        (qp, qs), (kp, ks), (vp, vs) = _rows(q, dtype, m, x if gate is None else 2 * x, gpu), _rows(k, dtype, m, self.width, gpu), _rows(v, dtype, m, self.width, gpu)
        if ks != vs:
            raise RuntimeError("the rows of k and v are %d and %d apart: one stride is needed" % (ks, vs))
        if not self.calls[5](self.p, layer, qp, kp, vp, dtype is self.bf16, qs, ks, n_head, _dense(wq, self.f32, self.hd, gpu), _dense(wk, self.f32, self.hd, gpu),
                             -1.0 if eps is None else eps, rope.p, _dense(pos, self.i32, m, gpu), _dense(slot, self.i32, m, gpu), m,
                             _dense(q_out, self.bf16 if q_bf16 else self.f32, m * x, gpu), q_bf16, _dense(gate, self.f32, m * x, gpu)):
            check(False, "q4_gpu_pages_prep")

    def fork(self, rows, src, dst, length, table):
        """request dst[i], which holds nothing, gets the first length[i] rows of request src[i]; rows[dst[i]] becomes length[i]"""
        i, gpu, (n, stride), m = self.i32, self.gpu, table.shape, src.shape[0]
        if not self.calls[6](self.p, self.shared, _dense(rows, i, n, gpu), n, _dense(src, i, m, gpu), _dense(dst, i, m, gpu), _dense(length, i, m, gpu), m,
                             _dense(table, i, n * stride, gpu), stride):
            check(False, "q4_gpu_pages_fork")

    def release(self, rows, keep, table):
        """request r keeps the first keep[r] of its rows, which rows[r] becomes; pages go back with their last holder"""
        i, gpu, (n, stride) = self.i32, self.gpu, table.shape
        if not self.calls[7](self.p, self.shared, _dense(rows, i, n, gpu), _dense(keep, i, n, gpu), n, _dense(table, i, n * stride, gpu), stride):
            check(False, "q4_gpu_pages_release")

    def compact(self, rows, table, number):
        """the pages in use to the low end of the pool; number [n_pages] gets every page's new one (-1: free).  rows and table None: the tables are renamed by the host"""
        i, gpu = self.i32, self.gpu
        n, stride = (0, 0) if table is None else table.shape
        if (rows is None) != (table is None):
            raise RuntimeError("a table and what its requests hold go together")
        if not self.calls[8](self.p, self.shared, _dense(rows, i, n, gpu), n, _dense(table, i, n * stride, gpu), stride, _dense(number, i, self.n_pages, gpu)):
            check(False, "q4_gpu_pages_compact")


def verify(logits, token, start, u_accept, u_next, accepted, next, draft=None, temp=None, logp=None, rows=None, keep=None):
    """drafted tokens held against the target's logits [n_tok][vocab] (fp32 or bf16, dense in its rows, as draft's), and the token behind the last one that is
    kept (q4_gpu_verify): token [n_tok] and start [n_req + 1] as the step was planned, u_accept [n_tok], u_next, accepted, next, temp, rows and keep [n_req], logp [n_tok]"""
    import torch
    L = load()
    gpu, (m, vocab), n, dtype, i, f = L.q4_gpu_device(), logits.shape, start.shape[0] - 1, logits.dtype, torch.int32, torch.float32
    if dtype is not f and dtype is not torch.bfloat16:
        raise RuntimeError("logits of %s are neither fp32 nor bf16" % dtype)
    (p, ld), (d, draft_ld) = _rows(logits, dtype, m, vocab, gpu), (None, 0) if draft is None else _rows(draft, dtype, m, vocab, gpu)
    if not L.q4_gpu_verify(p, dtype is torch.bfloat16, ld, d, draft_ld, vocab, _dense(token, i, m, gpu), _dense(start, i, n + 1, gpu), n, m, _dense(temp, f, n, gpu),
                           _dense(u_accept, f, m, gpu), _dense(u_next, f, n, gpu), _dense(accepted, i, n, gpu), _dense(next, i, n, gpu), _dense(logp, f, m, gpu),
                           _dense(rows, i, n, gpu), _dense(keep, i, n, gpu)):
        check(False, "q4_gpu_verify")
