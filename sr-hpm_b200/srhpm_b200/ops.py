"""Host-side operator layer of the B200 verify path, shaped like the ggml operators it replaces.

    Context.mul_mat(W, X)          ggml_mul_mat(W, X) with ne[1] = N = 1..16 on a GGUF-quantized W
                                   (reference: tensor_traits_srv::compute_forward, patch/srhpm.patch:6400-6611)
    Context.flash_attn_ext(...)    ggml_flash_attn_ext with 1..16 query rows over an f16 / q8_0 KV cache
                                   (reference: ggml_compute_forward_flash_attn_ext_gqa_small, patch/srhpm.patch:581-824)
    Context.flash_attn_ext_partial / flash_attn_merge
                                   the same attention split over KV token ranges: one (max, sum, acc) record set per
                                   range, merged after a gather (reference: its chunk records and their merge,
                                   patch/srhpm.patch:779-823, with devices as the chunks)
    Context.sample_and_accept_n()  greedy longest-prefix acceptance (reference: common_sampler_sample_and_accept_n,
                                   patch/srhpm.patch:1-37)
    Context.page_plan / rope_kv_paged / flash_attn_paged / adjust_logits / verify_sample
                                   a batch of sequences over a paged KV cache (f16, q8_0 or q4_0): the step's tables and
                                   slots, the store into pages, attention over them, penalties, biases and token masks
                                   on the logits, acceptance by sampling (no reference counterpart)
    Context.page_fork / page_copy / page_free / page_compact
                                   pages between steps: sequences that go on from others', whole-page copies in all
                                   layers, finished sequences' pages given back, pages in use moved together (no
                                   reference counterpart)

Tensors are torch tensors in device memory; torch only provides allocation and streams. Every compute call goes to
libsrhpm_b200.so through its C ABI; a missing library raises.
"""
import collections
import ctypes
import struct
import warnings

import numpy as np
import torch

from . import _lib as L


def _tensor_view(t, type_, ne, nb):
    v = L.SrhpmTensor()
    v.type = type_
    for i in range(4):
        v.ne[i] = ne[i] if i < len(ne) else 1
    last = nb[-1] * (ne[len(nb) - 1] if len(nb) else 1)
    for i in range(4):
        v.nb[i] = nb[i] if i < len(nb) else last
    v.data = t.data_ptr() if t is not None else 0
    return v


def f32_rows_view(x):
    """ggml view of a 2-D f32 tensor [rows, cols] (cols innermost): ne = [cols, rows]."""
    assert x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
    return _tensor_view(x, L.F32, [x.shape[1], x.shape[0]], [4, x.stride(0) * 4])


def _stream_ptr(stream):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


# cudaStream_t of a device's current stream (torch's own shortcut where it has one: the public way takes 2 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

PagePlan = collections.namedtuple("PagePlan", "q_start kv_len pos slots status n_taken")
PageFork = collections.namedtuple("PageFork", "src dst status n_taken")
PageMoves = collections.namedtuple("PageMoves", "src dst n_moves n_used")

# The calls of a serving step are short on the GPU, so their host side is kept short too: a view is the bytes of an
# srhpm_tensor (type, ne[4], nb[4], data), packed in one go.
_pack = struct.Struct("@iqqqqNNNNP").pack
_address = struct.Struct("@P")  # the last of them
assert struct.calcsize("@iqqqqNNNNP") == ctypes.sizeof(L.SrhpmTensor)


def _rows_2d(x, dtype, type_, what):
    """View of a 2-D tensor [rows, cols] of 4-byte values with contiguous rows: ne = [cols, rows]."""
    if x.dtype is not dtype or x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError(f"{what} must be {dtype} [rows, cols] with contiguous rows")
    r, c = x.shape
    nb = x.stride(0) * 4
    return _pack(type_, c, r, 1, 1, 4, nb, nb * r, nb * r, x.data_ptr())


def _head_rows(x, heads_first):
    """View of token rows [T, H, D] (f32 or f16, any strides of the first two): ne = [D, T, H], or [D, H, T]."""
    e = 2 if x.dtype is torch.float16 else 4 if x.dtype is torch.float32 else 0
    if e == 0 or x.dim() != 3 or x.stride(2) != 1:
        raise ValueError("rows must be f16 or f32 [T, H, D] with contiguous heads")
    T, H, D = x.shape
    a, b, _ = x.stride()
    a *= e
    b *= e
    t = L.F16 if e == 2 else L.F32
    if heads_first:
        return _pack(t, D, H, T, 1, e, b, a, a * T, x.data_ptr())
    return _pack(t, D, T, H, 1, e, a, b, a * T, x.data_ptr())


_BLOCK = {L.Q8_0: (34, 32), L.Q4_0: (18, 32)}  # bytes and values of a block


def _paged(c, kv_type):
    """View of a paged cache uint8 [pages, page_size, Hkv, row bytes]: ne = [D, page_size, Hkv, pages]."""
    if c.dtype is not torch.uint8 or c.dim() != 4 or c.stride(3) != 1:
        raise ValueError("a paged cache is uint8 [pages, page_size, Hkv, row bytes] with contiguous rows")
    n, P, Hkv, rowb = c.shape
    n3, n1, n2, _ = c.stride()
    size, blk = _BLOCK.get(kv_type, (2, 1))
    if rowb % size:
        raise ValueError("row bytes do not hold whole blocks of the cache type")
    return _pack(kv_type, rowb // size * blk, P, Hkv, n, size, n1, n2, n3, c.data_ptr())


def _pools(caches, kv_type):
    """Views of paged caches; those laid out like the first one differ from its view in the address alone."""
    if not caches:
        raise ValueError("no cache")
    first = caches[0]
    head, u8, shape, stride = _paged(first, kv_type)[:-_address.size], torch.uint8, first.shape, first.stride()
    return b"".join([head + _address.pack(c.data_ptr()) if c.shape == shape and c.stride() == stride and c.dtype is u8
                     else _paged(c, kv_type) for c in caches])


def _ints(t, dtype, n, what):
    """Address of a contiguous integer or f32 vector of at least n values."""
    if t.dtype is not dtype or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{what} must be a contiguous {dtype} vector of at least {n} values")
    return t.data_ptr()


def quantize_chunk(w, qtype):
    """Host weight quantizer: f32 [rows, K] (numpy or CPU torch) -> GGUF-packed bytes (numpy uint8, rows x row_size).
    ggml_quantize_chunk's contract (srhpm_quantize_chunk)."""
    lib = L.load()
    w = np.ascontiguousarray(np.asarray(w, dtype=np.float32))
    rows, K = w.shape
    rs = lib.srhpm_row_size(qtype, K)
    if rs == 0:
        raise ValueError(f"K={K} is not a multiple of the block size of {L.TYPE_NAMES.get(qtype, qtype)}")
    out = np.empty((rows, rs), dtype=np.uint8)
    n = lib.srhpm_quantize_chunk(qtype, w.ctypes.data, out.ctypes.data, 0, rows, K, None)
    if n != rows * rs:
        raise RuntimeError("srhpm_quantize_chunk failed")
    return out


def row_size(qtype, K):
    """Bytes of a row of K values of qtype (ggml_row_size)."""
    return int(L.load().srhpm_row_size(qtype, K))


def type_size(qtype):
    """Bytes of one block of qtype (ggml_type_size)."""
    return int(L.load().srhpm_type_size(qtype))


def blck_size(qtype):
    """Values per block of qtype (ggml_blck_size)."""
    return int(L.load().srhpm_blck_size(qtype))


class QuantTensor:
    """GGUF-packed weight rows in device memory: a ggml tensor of a quantized type with ne = [K, rows]."""

    def __init__(self, data, qtype, rows, K):
        lib = L.load()
        self.qtype, self.rows, self.K = qtype, rows, K
        self.row_bytes = lib.srhpm_row_size(qtype, K)
        if self.row_bytes == 0:
            raise ValueError("K is not a multiple of the block size")
        assert data.dtype == torch.uint8 and data.is_cuda and data.numel() >= rows * self.row_bytes
        self.data = data

    @classmethod
    def from_blocks(cls, blocks, qtype, rows, K, device="cuda"):
        # a read-only map of a GGUF file is fine here: the host tensor is only read by the copy to the device
        with warnings.catch_warnings():
            warnings.filterwarnings("ignore", message="The given NumPy array is not writable")
            t = torch.from_numpy(np.ascontiguousarray(blocks).reshape(-1)).to(device)
        return cls(t, qtype, rows, K)

    @classmethod
    def quantize(cls, w, qtype, device="cuda"):
        w = np.asarray(w, dtype=np.float32)
        return cls.from_blocks(quantize_chunk(w, qtype), qtype, w.shape[0], w.shape[1], device)

    def view(self):
        lib = L.load()
        return _tensor_view(self.data, self.qtype, [self.K, self.rows], [lib.srhpm_type_size(self.qtype),
                                                                         self.row_bytes])

    def row_slice(self, r0, r1):
        """Rows [r0, r1) as their own tensor (a view: the reference's CPU/GPU row split)."""
        sub = self.data[r0 * self.row_bytes:r1 * self.row_bytes]
        return QuantTensor(sub, self.qtype, r1 - r0, self.K)

    @property
    def nbytes(self):
        return self.rows * self.row_bytes


class Context:
    """srhpm_ctx of one device plus a cached work buffer."""

    def __init__(self, device=0):
        self.lib = L.load()
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        h = ctypes.c_void_p()
        L.check(self.lib.srhpm_ctx_create(self.device.index or 0, ctypes.byref(h)), "srhpm_ctx_create")
        self.handle = h
        self._work = None
        self._index = self.device.index or 0
        self._sizes = {}

    def close(self):
        if self.handle:
            self.lib.srhpm_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_q8_0_act_mode(self, mode):
        L.check(self.lib.srhpm_ctx_set_q8_0_act_mode(self.handle, mode), "set_q8_0_act_mode")

    def launch_count(self, reset=False):
        return int(self.lib.srhpm_ctx_launch_count(self.handle, 1 if reset else 0))

    def check(self):
        code = ctypes.c_int32(0)
        st = self.lib.srhpm_ctx_check(self.handle, ctypes.byref(code))
        if st != L.OK:
            raise L.SrhpmError(st, f"device status {code.value}", self.lib)

    def work(self, nbytes):
        if self._work is None or self._work.numel() < nbytes:
            self._work = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=self.device)
        return self._work

    # ---- small-batch quantized matmul -------------------------------------------------------------------------
    def mul_mat_work_size(self, W, X):
        wv, xv = W.view(), f32_rows_view(X)
        sz = ctypes.c_size_t()
        st = self.lib.srhpm_mul_mat_work_size(ctypes.byref(wv), ctypes.byref(xv), ctypes.byref(sz))
        return st, sz.value

    def mul_mat(self, W, X, out=None, stream=None, work=None, fused_quant=False):
        """Y[N, rows] = X[N, K] . W[rows, K]^T (ggml_mul_mat(W, X): dst ne = [rows, N]). fused_quant: one launch, the
        matmul grid quantizes its own activations (srhpm_mul_mat_fused_quant; bit-identical output)."""
        X = X if X.stride(-1) == 1 else X.contiguous()
        N = X.shape[0]
        if out is None:
            out = torch.empty((N, W.rows), dtype=torch.float32, device=X.device)
        wv, xv, yv = W.view(), f32_rows_view(X), f32_rows_view(out)
        st, ws = self.mul_mat_work_size(W, X)
        L.check(st, "srhpm_mul_mat_work_size")
        buf = work if work is not None else self.work(ws)
        fn = self.lib.srhpm_mul_mat_fused_quant if fused_quant else self.lib.srhpm_mul_mat
        L.check(fn(self.handle, ctypes.byref(wv), ctypes.byref(xv), ctypes.byref(yv), ctypes.c_void_p(buf.data_ptr()),
                   buf.numel(), _stream_ptr(stream)), "srhpm_mul_mat")
        return out

    def mul_mat_swiglu(self, W, gate, up, out=None, stream=None, work=None):
        """Y[N, rows] = (silu(gate) * up)[N, K] . W[rows, K]^T with the SwiGLU in the matmul grid's own prologue
        (srhpm_mul_mat_swiglu; gate and up of the same shape and row stride, e.g. the two halves of a gate|up
        product)."""
        N = gate.shape[0]
        if out is None:
            out = torch.empty((N, W.rows), dtype=torch.float32, device=gate.device)
        wv, gv, uv, yv = W.view(), f32_rows_view(gate), f32_rows_view(up), f32_rows_view(out)
        st, ws = self.mul_mat_work_size(W, gate)
        L.check(st, "srhpm_mul_mat_work_size")
        buf = work if work is not None else self.work(ws)
        L.check(self.lib.srhpm_mul_mat_swiglu(self.handle, ctypes.byref(wv), ctypes.byref(gv), ctypes.byref(uv),
                                              ctypes.byref(yv), ctypes.c_void_p(buf.data_ptr()), buf.numel(),
                                              _stream_ptr(stream)), "srhpm_mul_mat_swiglu")
        return out

    def prepare_mul_mat(self, W, X, Y, work, fused_quant=False):
        """A zero-argument callable that issues srhpm_mul_mat(W, X) -> Y on the current stream with prebuilt
        arguments (the per-call host cost is one ctypes call); usable under CUDA-graph capture, since the call
        allocates nothing."""
        wv, xv, yv = W.view(), f32_rows_view(X), f32_rows_view(Y)
        st, ws = self.mul_mat_work_size(W, X)
        L.check(st, "srhpm_mul_mat_work_size")
        if work.numel() < ws:
            raise ValueError("work buffer too small")
        fn, lib = (self.lib.srhpm_mul_mat_fused_quant if fused_quant else self.lib.srhpm_mul_mat), self.lib
        args = [self.handle, ctypes.byref(wv), ctypes.byref(xv), ctypes.byref(yv), ctypes.c_void_p(work.data_ptr()),
                work.numel()]
        keep = (wv, xv, yv, W, X, Y, work)

        def run():
            st = fn(*args, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            if st != L.OK:
                raise L.SrhpmError(st, "srhpm_mul_mat", lib)

        run.keep = keep
        return run

    def mul_mat_isums(self, W, X, stream=None):
        """Integer block sums of the matmul: isum, imin int32 [N, rows, nblk] (imin only for Q4_K / Q5_K)."""
        X = X.contiguous()
        N = X.shape[0]
        nblk = W.K // (32 if W.qtype == L.Q8_0 else 256)
        isum = torch.zeros((N, W.rows, nblk), dtype=torch.int32, device=X.device)
        imin = torch.zeros_like(isum)
        wv, xv = W.view(), f32_rows_view(X)
        st, ws = self.mul_mat_work_size(W, X)
        L.check(st, "srhpm_mul_mat_work_size")
        buf = self.work(ws)
        L.check(self.lib.srhpm_mul_mat_isums(self.handle, ctypes.byref(wv), ctypes.byref(xv),
                                             ctypes.c_void_p(isum.data_ptr()), ctypes.c_void_p(imin.data_ptr()),
                                             ctypes.c_void_p(buf.data_ptr()), buf.numel(), _stream_ptr(stream)),
                "srhpm_mul_mat_isums")
        return isum, imin

    # ---- multi-query attention (ggml_flash_attn_ext) -------------------------------------------------------------
    @staticmethod
    def _fa_views(q, k, v, kv_type, mask, sinks, out):
        """ggml views: q f32 [H, N, D] -> ne [D, N, H]; k / v uint8 [Hkv, L, row bytes] (any strides, rows
        contiguous) -> ne [D, L, Hkv]; mask f16 [N', L'] or [ne2, N', L'] -> ne [L', N', ne2]; sinks f32 [H];
        out f32 [N, H, DV] -> ne [DV, H, N]."""
        assert q.dtype == torch.float32 and q.dim() == 3 and q.stride(2) == 1
        H, N, D = q.shape
        tsz, blk = (34, 32) if kv_type == L.Q8_0 else (2, 1)
        views = [_tensor_view(q, L.F32, [D, N, H], [4, q.stride(1) * 4, q.stride(0) * 4])]
        for t in (k, v):
            assert t.dtype == torch.uint8 and t.dim() == 3 and t.stride(2) == 1
            Hkv, Lk, rowb = t.shape
            views.append(_tensor_view(t, kv_type, [rowb // tsz * blk, Lk, Hkv], [tsz, t.stride(1), t.stride(0)]))
        mv = None
        if mask is not None:
            assert mask.dtype == torch.float16 and mask.stride(-1) == 1
            m3 = mask if mask.dim() == 3 else mask.unsqueeze(0)
            mv = _tensor_view(m3, L.F16, [m3.shape[2], m3.shape[1], m3.shape[0]], [2, m3.stride(1) * 2, m3.stride(0) * 2])
        sv = None
        if sinks is not None:
            assert sinks.dtype == torch.float32 and sinks.dim() == 1 and sinks.stride(0) == 1
            sv = _tensor_view(sinks, L.F32, [sinks.shape[0]], [4])
        ov = None
        if out is not None:
            Nn, Hh, DV = out.shape
            ov = _tensor_view(out, L.F32, [DV, Hh, Nn], [4, out.stride(1) * 4, out.stride(0) * 4])
        return views[0], views[1], views[2], mv, sv, ov

    def flash_attn_ext_work_size(self, q, k, v, kv_type):
        qv, kvv, vv, _, _, _ = self._fa_views(q, k, v, kv_type, None, None, None)
        sz = ctypes.c_size_t()
        st = self.lib.srhpm_flash_attn_ext_work_size(self.handle, ctypes.byref(qv), ctypes.byref(kvv),
                                                     ctypes.byref(vv), ctypes.byref(sz))
        return st, sz.value

    def flash_attn_ext(self, q, k, v, kv_type, mask=None, sinks=None, scale=1.0, max_bias=0.0, softcap=0.0,
                       out=None, stream=None, work=None):
        """ggml_flash_attn_ext(q, k, v, mask, scale, max_bias, softcap) + sinks: out f32 [N, H, DV]."""
        H, N, D = q.shape
        DV = v.shape[2] // 34 * 32 if kv_type == L.Q8_0 else v.shape[2] // 2
        if out is None:
            out = torch.empty((N, H, DV), dtype=torch.float32, device=q.device)
        qv, kvv, vv, mv, sv, ov = self._fa_views(q, k, v, kv_type, mask, sinks, out)
        st, ws = self.flash_attn_ext_work_size(q, k, v, kv_type)
        L.check(st, "srhpm_flash_attn_ext_work_size")
        buf = work if work is not None else self.work(ws)
        L.check(self.lib.srhpm_flash_attn_ext(self.handle, ctypes.byref(qv), ctypes.byref(kvv), ctypes.byref(vv),
                                              ctypes.byref(mv) if mv is not None else None,
                                              ctypes.byref(sv) if sv is not None else None, scale, max_bias, softcap,
                                              ctypes.byref(ov), ctypes.c_void_p(buf.data_ptr()), buf.numel(),
                                              _stream_ptr(stream)), "srhpm_flash_attn_ext")
        return out

    # ---- attention split over the KV range across devices ------------------------------------------------------
    def flash_attn_part_size(self, H, N):
        """Bytes of one record set of srhpm_flash_attn_ext_partial for H heads and N query tokens."""
        return int(self.lib.srhpm_flash_attn_part_size(H, N))

    def flash_attn_ext_partial(self, q, k, v, kv_type, mask=None, scale=1.0, max_bias=0.0, softcap=0.0, out=None,
                               stream=None, work=None):
        """The record set of this KV range (k / v uint8 [Hkv, range tokens, row bytes], mask f16 [N', range tokens]
        or [ne2, N', range tokens]; a range of 0 tokens is allowed): uint8 [flash_attn_part_size(H, N)] on the
        device, for flash_attn_merge."""
        H, N, D = q.shape
        nbytes = self.flash_attn_part_size(H, N)
        if out is None:
            out = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        assert out.dtype == torch.uint8 and out.numel() >= nbytes and out.data_ptr() % 16 == 0
        qv, kvv, vv, mv, _, _ = self._fa_views(q, k, v, kv_type, mask, None, None)
        ws = 0
        if k.shape[1] > 0:
            st, ws = self.flash_attn_ext_work_size(q, k, v, kv_type)
            L.check(st, "srhpm_flash_attn_ext_work_size")
        buf = work if work is not None else self.work(ws)
        L.check(self.lib.srhpm_flash_attn_ext_partial(self.handle, ctypes.byref(qv), ctypes.byref(kvv),
                                                      ctypes.byref(vv), ctypes.byref(mv) if mv is not None else None,
                                                      scale, max_bias, softcap, ctypes.c_void_p(out.data_ptr()),
                                                      ctypes.c_void_p(buf.data_ptr()), buf.numel(),
                                                      _stream_ptr(stream)), "srhpm_flash_attn_ext_partial")
        return out

    def flash_attn_merge(self, parts, n_parts, H, N, sinks=None, out=None, stream=None):
        """Merge n_parts record sets stored one after another in `parts` (uint8, e.g. gathered from all devices in
        KV order), add the sinks and normalize: out f32 [N, H, 256], as flash_attn_ext over the whole range."""
        assert parts.dtype == torch.uint8 and parts.is_contiguous()
        assert parts.numel() >= n_parts * self.flash_attn_part_size(H, N)
        if out is None:
            out = torch.empty((N, H, 256), dtype=torch.float32, device=parts.device)
        ov = _tensor_view(out, L.F32, [out.shape[2], out.shape[1], out.shape[0]],
                          [4, out.stride(1) * 4, out.stride(0) * 4])
        sv = None
        if sinks is not None:
            assert sinks.dtype == torch.float32 and sinks.dim() == 1 and sinks.stride(0) == 1
            sv = _tensor_view(sinks, L.F32, [sinks.shape[0]], [4])
        L.check(self.lib.srhpm_flash_attn_merge(self.handle, ctypes.c_void_p(parts.data_ptr()), n_parts,
                                                ctypes.byref(sv) if sv is not None else None, ctypes.byref(ov),
                                                _stream_ptr(stream)), "srhpm_flash_attn_merge")
        return out

    def flash_attn_peer_buffer_size(self, H, N):
        """Bytes of one rank's buffer for flash_attn_merge_peers: the record set, then its receive area."""
        return int(self.lib.srhpm_flash_attn_peer_buffer_size(H, N))

    def flash_attn_merge_peers(self, peers, world, rank, epochs, H, N, sinks=None, out=None, stream=None):
        """srhpm_flash_attn_merge_peers: every rank's record set at the start of its own peer buffer (peers: int64
        device tensor of the world buffers' addresses on this device), exchanged as (value, epoch) words and merged in
        rank order; epochs: int32 [H * N] device counters, zero at the start. Returns out f32 [N, H, 256]."""
        if out is None:
            out = torch.empty((N, H, 256), dtype=torch.float32, device=peers.device)
        ov = _tensor_view(out, L.F32, [out.shape[2], out.shape[1], out.shape[0]],
                          [4, out.stride(1) * 4, out.stride(0) * 4])
        sv = None
        if sinks is not None:
            assert sinks.dtype == torch.float32 and sinks.dim() == 1 and sinks.stride(0) == 1
            sv = _tensor_view(sinks, L.F32, [sinks.shape[0]], [4])
        assert epochs.numel() >= H * N
        L.check(self.lib.srhpm_flash_attn_merge_peers(self.handle, ctypes.c_void_p(peers.data_ptr()), world, rank,
                                                      ctypes.c_void_p(epochs.data_ptr()),
                                                      ctypes.byref(sv) if sv is not None else None, ctypes.byref(ov),
                                                      _stream_ptr(stream)), "srhpm_flash_attn_merge_peers")
        return out

    # ---- greedy acceptance ------------------------------------------------------------------------------------------
    def sample_and_accept_n(self, logits, draft, relax=0.0, stream=None, work=None):
        """common_sampler_sample_and_accept_n (greedy): logits f32 [>= n_draft + 1, n_vocab] (rows = positions),
        draft int32 [n_draft] on the device -> (ids int32 [n_draft + 1], n int32 [1]) on the device; the emitted ids
        are ids[:n]."""
        assert logits.dtype == torch.float32 and logits.dim() == 2 and logits.stride(1) == 1
        n_draft = int(draft.numel())
        lv = _tensor_view(logits, L.F32, [logits.shape[1], logits.shape[0]], [4, logits.stride(0) * 4])
        sz = ctypes.c_size_t()
        L.check(self.lib.srhpm_verify_accept_work_size(self.handle, ctypes.byref(lv), ctypes.byref(sz)),
                "srhpm_verify_accept_work_size")
        buf = work if work is not None else self.work(sz.value)
        ids = torch.empty(n_draft + 1, dtype=torch.int32, device=logits.device)
        n = torch.empty(1, dtype=torch.int32, device=logits.device)
        d = draft.to(torch.int32).contiguous() if n_draft else None
        L.check(self.lib.srhpm_verify_accept(self.handle, ctypes.byref(lv),
                                             ctypes.c_void_p(d.data_ptr()) if d is not None else None, n_draft,
                                             relax, ctypes.c_void_p(ids.data_ptr()), ctypes.c_void_p(n.data_ptr()),
                                             ctypes.c_void_p(buf.data_ptr()), buf.numel(), _stream_ptr(stream)),
                "srhpm_verify_accept")
        return ids, n

    def argmax_shard(self, logits, vocab_offset, draft=None, stream=None, work=None):
        """Per-row record of a vocabulary shard: uint8 [rows, 16] (srhpm_argmax_record) on the device."""
        assert logits.dtype == torch.float32 and logits.dim() == 2 and logits.stride(1) == 1
        rows = logits.shape[0]
        lv = _tensor_view(logits, L.F32, [logits.shape[1], rows], [4, logits.stride(0) * 4])
        sz = ctypes.c_size_t()
        L.check(self.lib.srhpm_verify_accept_work_size(self.handle, ctypes.byref(lv), ctypes.byref(sz)),
                "srhpm_verify_accept_work_size")
        buf = work if work is not None else self.work(sz.value)
        rec = torch.empty((rows, 16), dtype=torch.uint8, device=logits.device)
        n_draft = int(draft.numel()) if draft is not None else 0
        d = draft.to(torch.int32).contiguous() if n_draft else None
        L.check(self.lib.srhpm_argmax_shard(self.handle, ctypes.byref(lv), vocab_offset,
                                            ctypes.c_void_p(d.data_ptr()) if d is not None else None, n_draft,
                                            ctypes.c_void_p(rec.data_ptr()), ctypes.c_void_p(buf.data_ptr()),
                                            buf.numel(), _stream_ptr(stream)), "srhpm_argmax_shard")
        return rec

    def accept_merge(self, recs, draft, relax=0.0, stream=None):
        """recs uint8 [n_shards, rows, 16] (argmax_shard outputs in vocabulary order) -> (ids, n) as
        sample_and_accept_n."""
        recs = recs.contiguous()
        n_shards, rows = recs.shape[0], recs.shape[1]
        n_draft = int(draft.numel())
        ids = torch.empty(n_draft + 1, dtype=torch.int32, device=recs.device)
        n = torch.empty(1, dtype=torch.int32, device=recs.device)
        d = draft.to(torch.int32).contiguous() if n_draft else None
        L.check(self.lib.srhpm_accept_merge(self.handle, ctypes.c_void_p(recs.data_ptr()), n_shards, rows,
                                            ctypes.c_void_p(d.data_ptr()) if d is not None else None, n_draft, relax,
                                            ctypes.c_void_p(ids.data_ptr()), ctypes.c_void_p(n.data_ptr()),
                                            _stream_ptr(stream)), "srhpm_accept_merge")
        return ids, n

    # ---- a batch of sequences over a paged KV cache --------------------------------------------------------------
    # Scratch and new outputs of these calls come from torch's allocator on the call's stream, call by call: calls on
    # several streams never share a buffer, and a captured graph keeps its own.
    def _on_device(self, *tensors):
        for t in tensors:
            if t is not None and t.get_device() != self._index:
                raise ValueError(f"a tensor on {t.device} given to a context of cuda:{self._index}")

    def _new(self, shape, dtype, stream):
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def _call(self, fn, what, stream, *args):
        """One C-ABI call on `stream` (the current stream of the context's device if None)."""
        s = _raw_stream(self._index) if stream is None else stream.cuda_stream
        if torch.cuda.current_device() == self._index:
            st = fn(self.handle, *args, s)
        else:
            with torch.cuda.device(self.device):
                st = fn(self.handle, *args, s)
        if st != L.OK:
            raise L.SrhpmError(st, what, self.lib)

    def _scratch(self, fn, what, key, stream, *args):
        """Work buffer of a call; its size goes by the shapes in `key` alone and is asked for once for each."""
        n = self._sizes.get(key)
        if n is None:
            sz = ctypes.c_size_t()
            L.check(fn(self.handle, *args, ctypes.byref(sz)), what)
            n = self._sizes[key] = max(sz.value, 16)
        return self._new(n, torch.uint8, stream)

    def page_plan(self, n_past, n_new, block_table, free_pages, page_size, n_rows, free_head=None, out=None,
                  stream=None, n_held=None):
        """Tables and slots of a step (srhpm_page_plan): n_past, n_new int32 [S]; block_table int32 [S, entries] (new
        entries are written into it); free_pages int32 [F], taken from free_head (int32 [1], 0 if None); n_held int32 [S]:
        pages that a row names already, if more than n_past fills (after rejected tokens, torch.maximum(n_held,
        (kv_len + page_size - 1) // page_size) of the step before). Returns a
        PagePlan: q_start int32 [S + 1], kv_len int32 [S], pos int32 [n_rows], slots int64 [n_rows], status int32 [S],
        n_taken int32 [1] (`out`: one to write into, which shares no memory with the inputs: not the plan whose kv_len is
        this step's n_past)."""
        S = n_past.numel()
        self._on_device(n_past, n_new, block_table, free_pages, free_head, n_held)
        i32 = torch.int32
        if out is None:
            at = self._new(3 * S + 2 + n_rows, i32, stream)
            q, k, st, nt, pos = at.split_with_sizes((S + 1, S, S, 1, n_rows))
            out = PagePlan(q, k, pos, self._new(n_rows, torch.int64, stream), st, nt)
            p = at.data_ptr()
            ptrs = (p, p + 4 * (S + 1), p + 4 * (3 * S + 2), out.slots.data_ptr(), p + 4 * (2 * S + 1),
                    p + 4 * (3 * S + 1))
        else:
            self._on_device(*out)
            ptrs = (_ints(out.q_start, i32, S + 1, "q_start"), _ints(out.kv_len, i32, S, "kv_len"),
                    _ints(out.pos, i32, n_rows, "pos"), _ints(out.slots, torch.int64, n_rows, "slots"),
                    _ints(out.status, i32, S, "status"), _ints(out.n_taken, i32, 1, "n_taken"))
        self._call(self.lib.srhpm_page_plan, "srhpm_page_plan", stream, _ints(n_past, i32, S, "n_past"),
                   _ints(n_new, i32, S, "n_new"), None if n_held is None else _ints(n_held, i32, S, "n_held"), S,
                   page_size, _rows_2d(block_table, i32, L.I32, "block_table"),
                   _ints(free_pages, i32, 0, "free_pages"), free_pages.numel(),
                   None if free_head is None else _ints(free_head, i32, 1, "free_head"), n_rows, *ptrs)
        return out

    def rope_kv_paged(self, qkv, pos, slots, k_cache, v_cache, kv_type, q_out, theta_base=1e6, stream=None):
        """RoPE of fused rows qkv f32 [n, (H + 2 Hkv) D] (only read) at pos int32 [n]: turned queries into q_out [n, H,
        D] (f16 or f32), turned keys and values into the cache rows of slots int64 [n] (srhpm_rope_kv_paged). Caches:
        uint8 [pages, page_size, Hkv, row bytes]. Returns q_out."""
        n = qkv.shape[0]
        self._on_device(qkv, pos, slots, k_cache, v_cache, q_out)
        self._call(self.lib.srhpm_rope_kv_paged, "srhpm_rope_kv_paged", stream,
                   _rows_2d(qkv, torch.float32, L.F32, "qkv"), q_out.shape[1], k_cache.shape[2],
                   _ints(pos, torch.int32, n, "pos"), _ints(slots, torch.int64, n, "slots"), theta_base,
                   _head_rows(q_out, False), _paged(k_cache, kv_type), _paged(v_cache, kv_type))
        return q_out

    def flash_attn_paged(self, q, k_cache, v_cache, kv_type, block_table, q_start, kv_len, scale=1.0, softcap=0.0,
                         window=0, sinks=None, out=None, stream=None, work=None):
        """Causal attention of the new rows q [T, H, D] (f16 or f32) of S sequences over their pages
        (srhpm_flash_attn_paged): block_table int32 [S, entries], q_start int32 [S + 1], kv_len int32 [S] as page_plan
        gives them; window > 0: only the last `window` positions. Returns out [T, H, D] of q's type (padding rows as
        they were; of a new tensor: anything)."""
        S = block_table.shape[0]
        if out is None:
            out = self._new(q.shape, q.dtype, stream)
        self._on_device(q, k_cache, v_cache, block_table, q_start, kv_len, sinks, out, work)
        qv, kv = _head_rows(q, False), _paged(k_cache, kv_type)
        if work is None:
            work = self._scratch(self.lib.srhpm_flash_attn_paged_work_size, "srhpm_flash_attn_paged_work_size",
                                 ("fa", q.shape, q.dtype, k_cache.shape, kv_type, S), stream, qv, kv, S)
        sv = None
        if sinks is not None:
            at = _ints(sinks, torch.float32, q.shape[1], "sinks")
            sv = _pack(L.F32, sinks.shape[0], 1, 1, 1, 4, 4, 4, 4, at)
        self._call(self.lib.srhpm_flash_attn_paged, "srhpm_flash_attn_paged", stream, qv, kv, _paged(v_cache, kv_type),
                   _rows_2d(block_table, torch.int32, L.I32, "block_table"), _ints(q_start, torch.int32, S + 1, "q_start"),
                   _ints(kv_len, torch.int32, S, "kv_len"), sv, scale, softcap, window, _head_rows(out, True),
                   work.data_ptr(), work.numel())
        return out

    def page_fork(self, parent, child, n_keep, block_table, page_refs, free_pages, page_size, free_head=None, out=None,
                  stream=None):
        """New sequences that begin with the first n_keep[i] tokens of others (srhpm_page_fork): table row child[i] gets
        the pages of row parent[i], whole ones shared (counted in page_refs int32 [pages]: holders beyond the first), a
        partly filled one replaced by a page from free_pages (as in page_plan). parent, child, n_keep int32 [n].
        Returns a PageFork: src, dst int32 [n] (the copies still to be made with page_copy; -1: none), status int32 [n],
        n_taken int32 [1] (`out`: one to write into)."""
        n, i32 = parent.numel(), torch.int32
        self._on_device(parent, child, n_keep, block_table, page_refs, free_pages, free_head)
        if out is None:
            out = PageFork(*self._new(3 * n + 1, i32, stream).split_with_sizes((n, n, n, 1)))
        else:
            self._on_device(*out)
        self._call(self.lib.srhpm_page_fork, "srhpm_page_fork", stream, _ints(parent, i32, n, "parent"),
                   _ints(child, i32, n, "child"), _ints(n_keep, i32, n, "n_keep"), n, page_size,
                   _rows_2d(block_table, i32, L.I32, "block_table"), _ints(page_refs, i32, 1, "page_refs"),
                   page_refs.numel(), _ints(free_pages, i32, 0, "free_pages"), free_pages.numel(),
                   None if free_head is None else _ints(free_head, i32, 1, "free_head"), _ints(out.src, i32, n, "src"),
                   _ints(out.dst, i32, n, "dst"), _ints(out.status, i32, n, "status"),
                   _ints(out.n_taken, i32, 1, "n_taken"))
        return out

    def page_copy(self, caches, kv_type, src, dst, n_moves=None, stream=None):
        """Pages src[i] copied to dst[i] (int32 [n]; no page: nothing) in every pool of `caches`, a list of uint8 [pages,
        page_size, Hkv, row bytes] of one shape and layout, in one launch (srhpm_page_copy). n_moves int32 [1]: only that many."""
        self._on_device(src, dst, n_moves, *caches)
        n = src.numel()
        self._call(self.lib.srhpm_page_copy, "srhpm_page_copy", stream, _pools(caches, kv_type),
                   len(caches), _ints(src, torch.int32, n, "src"), _ints(dst, torch.int32, n, "dst"), n,
                   None if n_moves is None else _ints(n_moves, torch.int32, 1, "n_moves"))

    def page_free(self, rows, begin, end, block_table, page_refs, free_pages, free_head, out=None, stream=None):
        """Entries begin[i] .. end[i] - 1 of table rows rows[i] given up (int32 [n]; begin None: 0): they become -1, and pages that no
        sequence holds any more go onto the free list in front of free_head, in the order of their numbers
        (srhpm_page_free). Returns n_freed int32 [1] (`out`: one to write into): the next head is free_head - n_freed."""
        n, i32 = rows.numel(), torch.int32
        self._on_device(rows, begin, end, block_table, page_refs, free_pages, free_head, out)
        if out is None:
            out = self._new(1, i32, stream)
        self._call(self.lib.srhpm_page_free, "srhpm_page_free", stream, _ints(rows, i32, n, "rows"),
                   None if begin is None else _ints(begin, i32, n, "begin"), _ints(end, i32, n, "end"), n,
                   _rows_2d(block_table, i32, L.I32, "block_table"), _ints(page_refs, i32, 1, "page_refs"),
                   page_refs.numel(), _ints(free_pages, i32, 0, "free_pages"), free_pages.numel(),
                   _ints(free_head, i32, 1, "free_head"), _ints(out, i32, 1, "n_freed"))
        return out

    def page_compact(self, block_table, n_held, page_refs, free_pages, out=None, stream=None):
        """The pages that the first n_held[s] entries of the table's rows name get the lowest numbers (srhpm_page_compact):
        table, page_refs int32 [pages] and free_pages int32 [pages] are rewritten, and page_copy has still to move the bytes. Returns a
        PageMoves: src, dst int32 [pages // 2], n_moves, n_used int32 [1]; the free list's head is n_used from here on
        (`out`: (src, dst) to write into; entries behind n_moves stay as they are)."""
        n, i32 = page_refs.numel(), torch.int32
        self._on_device(block_table, n_held, page_refs, free_pages)
        if out is None:
            src, dst, count = self._new(2 * (n // 2) + 2, i32, stream).split_with_sizes((n // 2, n // 2, 2))
        else:
            self._on_device(*out)
            (src, dst), count = out, self._new(2, i32, stream)
        moves = PageMoves(src, dst, count[:1], count[1:])
        self._call(self.lib.srhpm_page_compact, "srhpm_page_compact", stream,
                   _rows_2d(block_table, i32, L.I32, "block_table"), _ints(n_held, i32, block_table.shape[0], "n_held"),
                   _ints(page_refs, i32, n, "page_refs"), n, _ints(free_pages, i32, n, "free_pages"),
                   _ints(src, i32, n // 2, "src"), _ints(dst, i32, n // 2, "dst"), count.data_ptr(), count.data_ptr() + 4)
        return moves

    def adjust_logits(self, logits, ids, q_start, history=None, n_history=None, last_n=None, repeat=None, frequency=None,
                      presence=None, bias=None, mask=None, mask_row=None, out=None, stream=None):
        """Rules on the logits f32 [T, V] of a step's rows before verify_sample (srhpm_adjust_logits): biases of tokens (bias:
        (starts int32 [S + 1], tokens int32, values f32)), penalties for the tokens in each row's window, the last
        last_n[s] (int32 [S]; negative or None: all) of history int32 [S, capacity] (n_history int32 [S] of them) and the sequence's rows up to this one in ids int32 [T]: repeat,
        frequency, presence f32 [S] or None; and masks int32 [n, >= ceil(V / 32)] with a bit per allowed token, row r's
        being mask_row[r] (int32 [T]; negative: none; None: r). Returns out (`out`: logits itself, or a tensor that
        shares nothing with them; None: a new one). Padding rows stay as they are."""
        T, S, i32, f32 = logits.shape[0], q_start.numel() - 1, torch.int32, torch.float32
        if out is None:
            out = self._new(logits.shape, f32, stream)
        if mask_row is not None and mask is None:
            raise ValueError("mask_row without a mask")
        starts, tokens, values = (None, None, None) if bias is None else bias
        self._on_device(logits, ids, q_start, history, n_history, last_n, repeat, frequency, presence, starts, tokens, values,
                        mask, mask_row, out)

        def vec(t, dtype, n, what):
            return None if t is None else _ints(t, dtype, n, what)

        nb = 0 if bias is None else tokens.numel()
        self._call(self.lib.srhpm_adjust_logits, "srhpm_adjust_logits", stream, _rows_2d(logits, f32, L.F32, "logits"),
                   _ints(ids, i32, T, "ids"), _ints(q_start, i32, S + 1, "q_start"), S,
                   None if history is None else _rows_2d(history, i32, L.I32, "history"), vec(n_history, i32, S, "n_history"),
                   vec(last_n, i32, S, "last_n"), vec(repeat, f32, S, "repeat"), vec(frequency, f32, S, "frequency"),
                   vec(presence, f32, S, "presence"), vec(starts, i32, S + 1, "bias starts"), vec(tokens, i32, nb, "bias tokens"),
                   vec(values, f32, nb, "bias values"), nb, None if mask is None else _rows_2d(mask, i32, L.I32, "mask"),
                   vec(mask_row, i32, T, "mask_row"), _rows_2d(out, f32, L.F32, "out"))
        return out

    def verify_sample(self, logits, ids, q_start, u_accept, u_sample, draft_probs=None, temperature=None, out=None,
                      stream=None, work=None):
        """Acceptance of drafted tokens by sampling (srhpm_verify_sample): logits f32 [T, V] of the step's rows, ids
        int32 [T] its input tokens (the drafted token of row r is ids[r + 1]), q_start int32 [S + 1], u_accept f32 [T],
        u_sample f32 [S], draft_probs f32 [T, V] or None (a drafter without distributions), temperature f32 [S] or
        None. Returns (out_ids int32 [T], out_n int32 [S], p_draft f32 [T]); sequence s emitted
        out_ids[q_start[s] : q_start[s] + out_n[s]]. `out`: three to write into, which share no memory with the inputs."""
        T, S = logits.shape[0], q_start.numel() - 1
        self._on_device(logits, ids, q_start, u_accept, u_sample, draft_probs, temperature, work)
        i32, f32 = torch.int32, torch.float32
        if out is None:
            out = (self._new(T, i32, stream), self._new(S, i32, stream), self._new(T, f32, stream))
        else:
            self._on_device(*out)
        lv = _rows_2d(logits, f32, L.F32, "logits")
        if work is None:
            work = self._scratch(self.lib.srhpm_verify_sample_work_size, "srhpm_verify_sample_work_size",
                                 ("vs", logits.shape, S), stream, lv, S)
        self._call(self.lib.srhpm_verify_sample, "srhpm_verify_sample", stream, lv, _ints(ids, i32, T, "ids"),
                   _ints(q_start, i32, S + 1, "q_start"), S,
                   None if draft_probs is None else _rows_2d(draft_probs, f32, L.F32, "draft_probs"),
                   None if temperature is None else _ints(temperature, f32, S, "temperature"),
                   _ints(u_accept, f32, T, "u_accept"), _ints(u_sample, f32, S, "u_sample"),
                   _ints(out[0], i32, T, "out_ids"), _ints(out[1], i32, S, "out_n"),
                   None if out[2] is None else _ints(out[2], f32, T, "p_draft"), work.data_ptr(), work.numel())
        return out

    def quantize_rows_q8_K(self, X, stream=None):
        X = X.contiguous()
        N, K = X.shape
        q = torch.empty((N, K), dtype=torch.int8, device=X.device)
        d = torch.empty((N, K // 256), dtype=torch.float32, device=X.device)
        b32 = torch.empty((N, K // 32), dtype=torch.int16, device=X.device)
        b16 = torch.empty((N, K // 16), dtype=torch.int16, device=X.device)
        xv = f32_rows_view(X)
        L.check(self.lib.srhpm_quantize_rows_q8_K(self.handle, ctypes.byref(xv), ctypes.c_void_p(q.data_ptr()),
                                                  ctypes.c_void_p(d.data_ptr()), ctypes.c_void_p(b32.data_ptr()),
                                                  ctypes.c_void_p(b16.data_ptr()), _stream_ptr(stream)),
                "srhpm_quantize_rows_q8_K")
        return q, d, b32, b16

    def quantize_rows_q8_0(self, X, stream=None):
        X = X.contiguous()
        N, K = X.shape
        out = torch.empty((N, (K // 32) * 34), dtype=torch.uint8, device=X.device)
        xv = f32_rows_view(X)
        L.check(self.lib.srhpm_quantize_rows_q8_0(self.handle, ctypes.byref(xv), ctypes.c_void_p(out.data_ptr()),
                                                  _stream_ptr(stream)), "srhpm_quantize_rows_q8_0")
        return out
