"""Python host side of libsfbert_b200.so: a ctypes binding of the C ABI (include/sfbert_b200.h)
plus thin helpers that mirror the reference's operator surface (blocksparse.h,
fusion_blocksparse.h) on torch tensors.  torch is used for device memory and streams only;
every operator below runs a hand-written sm_100a kernel from the shared library, and the import
fails loudly when the library is missing -- there is no fallback.  The operators' checks, output
allocations and calls are in C++ (csrc/host.cpp, the _host module): a call through ctypes took
17-20 us of host time, more than most small kernels run."""
import ctypes as C
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
# SFBERT_B200_LIB selects another build of the same library (e.g. an instrumented one)
LIB_PATH = os.environ.get("SFBERT_B200_LIB") or os.path.join(_HERE, "libsfbert_b200.so")

F32, BF16, F16 = 0, 1, 2
LAYOUT_FULL, LAYOUT_FIXED, LAYOUT_STRIDE, LAYOUT_SAWTOOTH, LAYOUT_LOCAL, LAYOUT_BIGBIRD = range(6)
MASK_ALL, MASK_CAUSAL_DIAG, MASK_CAUSAL_ALL, MASK_LOCAL = range(4)
NT_OP, NN_OP, TN_OP = 0, 1, 2
ACT_NONE, ACT_GELU = 0, 1

# every symbol include/sfbert_b200.h declares
SYMBOLS = [
    "sfb_last_error", "sfb_version", "sfb_layout_generate", "sfb_lut_count", "sfb_lut_build", "sfb_mask_pack",
    "sfb_magicu64", "sfb_bst_sgemm_nt", "sfb_masked_softmax", "sfb_bst_sgemm_xn", "sfb_fused_sddmm_softmax",
    "sfb_fused_attention", "sfb_bias_residual_layernorm", "sfb_device_status", "sfb_bias_gelu", "sfb_lut_build_tn",
    "sfb_masked_softmax_grad", "sfb_linear", "sfb_linear_nt", "sfb_embedding", "sfb_csr_from_layout",
    "sfb_csr_attention", "sfb_rowdot", "sfb_fused_sddmm_softmax_grad", "sfb_fused_attention_slice", "sfb_device_status_clear",
    "sfb_linear_residual", "sfb_attention_backward", "sfb_csr_workspace",
    "sfb_csr_attention_planned", "sfb_token_logprobs", "sfb_token_logprobs_grad", "sfb_distill_topk", "sfb_distill_topk_grad",
    "sfb_linear_logprobs", "sfb_linear_logprobs_workspace", "sfb_fused_attention_stats", "sfb_attention_backward_recompute",
    "sfb_attention_backward_workspace", "sfb_embedding_scaled", "sfb_embedding_grad", "sfb_embedding_grad_workspace", "sfb_grad_norm",
    "sfb_clip_grad_norm", "sfb_clip_grad_norm_workspace",
]

if not os.path.exists(LIB_PATH):
    raise ImportError("%s is missing: build it with `make -C %s/csrc` (needs nvcc, sm_100a)" % (LIB_PATH, _HERE))
if not os.path.exists(os.path.join(_HERE, "_host.so")):
    raise ImportError("%s/_host.so is missing: build it with `make -C %s/csrc` (needs g++ and torch's headers)" % (_HERE, _HERE))
lib = C.CDLL(LIB_PATH)
lib.sfb_last_error.restype = C.c_char_p
for _name in SYMBOLS:
    getattr(lib, _name)

from . import _host  # noqa: E402

_host.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in _host.wanted().split()})
SfbError = _host.SfbError

# The signatures of the C ABI, for programs that call `lib` themselves: without them ctypes would pass a pointer given as a
# plain integer as 32 bits.  The operators below go through _host and need them only where they call `lib`.
_u32, _i32, _u64, _f32, _vp = C.c_uint32, C.c_int, C.c_uint64, C.c_float, C.c_void_p
lib.sfb_layout_generate.argtypes = [_vp, _vp, _u32, _u32, _i32, _u32, _u32, _u32, _u32, _i32, _u64]
lib.sfb_lut_count.argtypes = [_vp, _vp, _u32, _u32, _vp]
lib.sfb_lut_build.argtypes = [_vp, _vp, _u32, _u32, _u32, _vp, _vp, _vp, _vp, _vp]
lib.sfb_mask_pack.argtypes = [_vp, _vp, _u32, _u32, _u32, _i32, _u32, _vp, _vp]
lib.sfb_magicu64.argtypes = [_u32, C.POINTER(_u32), C.POINTER(_u32)]
lib.sfb_magicu64.restype = None
lib.sfb_bst_sgemm_nt.argtypes = [_vp, _vp, _vp, _vp, _vp, _i32, _i32] + [_u32] * 9
lib.sfb_masked_softmax.argtypes = [_vp, _vp, _vp, _vp, _vp, _i32, _i32] + [_u32] * 9 + [_f32]
lib.sfb_bst_sgemm_xn.argtypes = [_vp, _vp, _vp, _vp, _vp, _i32, _i32] + [_u32] * 13
lib.sfb_lut_build_tn.argtypes = [_vp, _vp, _u32, _u32, _u32, _vp, _vp, _vp]
lib.sfb_masked_softmax_grad.argtypes = [_vp, _vp, _vp, _vp, _vp, _i32] + [_u32] * 8 + [_f32]
lib.sfb_linear.argtypes = [_vp, _vp, _vp, _vp, _vp, _u32, _u32, _u32, _i32, _i32]
lib.sfb_linear_nt.argtypes = [_vp, _vp, _vp, _vp, _vp, _u32, _u32, _u32, _i32, _i32]
lib.sfb_embedding.argtypes = [_vp, _vp, _vp, _vp, _vp, _u32, _u32, _u32, _u32, _i32, _vp]
lib.sfb_csr_from_layout.argtypes = [_vp, _vp, _u32, _u32, _vp, _vp]
lib.sfb_rowdot.argtypes = [_vp, _vp, _vp, _vp, _u64, _u32, _i32]
lib.sfb_fused_sddmm_softmax_grad.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32] + [_u32] * 8 + [_f32]
lib.sfb_csr_attention.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _u32, _u32, _u32, _u32, _f32, _vp]
lib.sfb_fused_sddmm_softmax.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32] + [_u32] * 10 + [_f32]
lib.sfb_fused_attention.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32] + [_u32] * 9 + [_f32, _u32]
lib.sfb_fused_attention_slice.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32] + [_u32] * 9 + [_f32, _u32, _u64, _u64]
lib.sfb_bias_residual_layernorm.argtypes = [_vp] * 10 + [_u32, _u32, _i32]
lib.sfb_device_status.argtypes = [C.POINTER(_u32)]
lib.sfb_bias_gelu.argtypes = [_vp, _vp, _vp, _vp, _u32, _u32, _i32]
lib.sfb_linear_residual.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _u32, _u32, _u32, _i32]
lib.sfb_attention_backward.argtypes = [_vp] * 13 + [_i32] + [_u32] * 10 + [_f32]
lib.sfb_csr_workspace.argtypes = [_u32, _u32]
lib.sfb_csr_workspace.restype = _u64
lib.sfb_csr_attention_planned.argtypes = [_vp, _vp, _vp, _u32, _vp, _vp, _vp, _vp, _i32, _u32, _u32, _u32, _u32, _f32, _vp, _vp]
lib.sfb_token_logprobs.argtypes = [_vp, _vp, _u64, _vp, _u32, _u32, _i32, _f32] + [_vp] * 5 + [_u32, _vp]
lib.sfb_token_logprobs_grad.argtypes = [_vp, _vp, _u64] + [_vp] * 6 + [_u64, _u32, _u32, _u32, _i32, _f32]
lib.sfb_distill_topk.argtypes = [_vp, _vp, _u64, _vp, _vp, _u32, _u32, _u32, _i32, _f32, _i32, _vp, _vp, _vp]
lib.sfb_distill_topk_grad.argtypes = [_vp, _vp, _u64] + [_vp] * 8 + [_u64, _u32, _u32, _u32, _u32, _i32, _f32, _i32]

lib.sfb_linear_logprobs_workspace.argtypes = [_u32, _u32]
lib.sfb_linear_logprobs_workspace.restype = _u64
lib.sfb_linear_logprobs.argtypes = [_vp] * 5 + [_u32, _u32, _u32, _i32, _f32] + [_vp] * 5

lib.sfb_fused_attention_stats.argtypes = [_vp] * 8 + [_i32] + [_u32] * 9 + [_f32, _u32, _u64, _u64]
lib.sfb_attention_backward_recompute.argtypes = [_vp] * 14 + [_i32] + [_u32] * 9 + [_f32, _u32, _u32] + [_u64] * 4 + [_vp, _u64]
lib.sfb_attention_backward_workspace.argtypes = [_i32] + [_u32] * 8 + [_i32]
lib.sfb_attention_backward_workspace.restype = _u64
lib.sfb_embedding_scaled.argtypes = [_vp] * 5 + [_u32] * 4 + [_i32, _f32, _vp]
lib.sfb_embedding_grad.argtypes = [_vp] * 5 + [_u32] * 4 + [_i32, _i32, _f32, _i32, _vp, _vp]
lib.sfb_embedding_grad_workspace.argtypes = [_u32] * 4
lib.sfb_embedding_grad_workspace.restype = _u64
lib.sfb_grad_norm.argtypes = [_vp, _u32, _vp, _vp, _vp, _f32, _vp, _vp]
lib.sfb_clip_grad_norm.argtypes = [_vp, _u32] + [_vp] * 5 + [_f32, _f32, _vp, _vp]
lib.sfb_clip_grad_norm_workspace.argtypes = [_u32]
lib.sfb_clip_grad_norm_workspace.restype = _u64


def device_status():
    """0 unless a kernel gave up on one of its bounded waits (synchronises with the device)."""
    v = _u32(0)
    _check(lib.sfb_device_status(C.byref(v)))
    return v.value


def device_status_clear():
    """Sets the status word back to 0 (synchronises with the device)."""
    _check(lib.sfb_device_status_clear())


def _check(rc):
    if rc != 0:
        raise SfbError(lib.sfb_last_error().decode())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def dtype_tag(t):
    return _DT[t.dtype]


def magicu64(d):
    """magicu64 of blocksparse.h:1016-1043."""
    m, s = _u32(0), _u32(0)
    lib.sfb_magicu64(d, C.byref(m), C.byref(s))
    return m.value, s.value


class BlockLayout:
    """A block layout and its look-up tables in device memory (what the reference's test programs
    build on the host and upload, stride_fusion_test.cu:48-227)."""

    def __init__(self, layout, block_size):
        assert layout.dtype == torch.uint8 and layout.dim() == 3 and layout.is_cuda
        self.layout = layout.contiguous()
        self.heads, self.nb, _ = layout.shape
        self.block_size = block_size
        dev = layout.device
        counts = torch.zeros(self.heads, dtype=torch.int32, device=dev)
        _check(lib.sfb_lut_count(_stream(), _p(self.layout), self.heads, self.nb, _p(counts)))
        counts = counts.cpu()  # the one host read: sizes the tables
        if int(counts.min()) != int(counts.max()):
            raise SfbError("heads have different block counts: %s" % counts.tolist())
        self.blocks = int(counts[0])
        self.nt_lut = torch.zeros(self.heads, self.blocks, 2, dtype=torch.int32, device=dev)
        self.nn_lut = torch.zeros(self.heads, self.nb + self.blocks, 2, dtype=torch.int32, device=dev)
        self.rblk_lut = torch.zeros(self.heads, self.blocks, 2, dtype=torch.int32, device=dev)
        nn_max = torch.zeros(1, dtype=torch.int32, device=dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        _check(lib.sfb_lut_build(_stream(), _p(self.layout), self.heads, self.nb, self.blocks, _p(self.nt_lut),
                                 _p(self.nn_lut), _p(self.rblk_lut), _p(nn_max), _p(status)))
        if int(status.item()) != 0:
            raise SfbError("sfb_lut_build: block count mismatch")
        self.nn_max = int(nn_max.item())
        self.mask_np = None
        self.mask_t = None
        self._tn = None

    def _build_tn(self):
        """The column-major LUT of the backward matmuls, built on first use."""
        if self._tn is None:
            dev = self.layout.device
            tn = torch.zeros(self.heads, self.nb + self.blocks, 2, dtype=torch.int32, device=dev)
            tn_max = torch.zeros(1, dtype=torch.int32, device=dev)
            status = torch.zeros(1, dtype=torch.int32, device=dev)
            _check(lib.sfb_lut_build_tn(_stream(), _p(self.layout), self.heads, self.nb, self.blocks, _p(tn), _p(tn_max),
                                        _p(status)))
            if int(status.item()) != 0:
                raise SfbError("sfb_lut_build_tn: block count mismatch")
            self._tn = (tn, int(tn_max.item()))
        return self._tn

    @property
    def tn_lut(self):
        return self._build_tn()[0]

    @property
    def tn_max(self):
        return self._build_tn()[1]

    @classmethod
    def generate(cls, kind, heads, nb, block_size, p0=0, p1=0, p2=0, p3=0, causal=0, seed=0, device="cuda"):
        lay = torch.empty(heads, nb, nb, dtype=torch.uint8, device=device)
        _check(lib.sfb_layout_generate(_stream(), _p(lay), heads, nb, kind, p0, p1, p2, p3, causal, seed))
        return cls(lay, block_size)

    def pack_mask(self, pred, ctx=0):
        wt = torch.int32 if self.block_size == 32 else torch.int64
        dev = self.layout.device
        self.mask_np = torch.zeros(self.heads, self.blocks, self.block_size, dtype=wt, device=dev)
        self.mask_t = torch.zeros(self.heads, self.block_size, self.blocks, dtype=wt, device=dev)
        _check(lib.sfb_mask_pack(_stream(), _p(self.nt_lut), self.heads, self.blocks, self.block_size, pred, ctx,
                                 _p(self.mask_np), _p(self.mask_t)))
        return self

    @property
    def nt_lut_dim(self):
        return self.blocks

    @property
    def nn_lut_dim(self):
        return self.blocks + self.nb


def bst_sgemm_nt(q, k, lay, out_dtype=torch.bfloat16):
    """S = Q.K^T on the kept blocks, unscaled (bst_sgemm_nt / bst_sgemm_nt_float, blocksparse.h:425,202)."""
    return _host.bst_sgemm_nt(q, k, lay, _DT[out_dtype])


def masked_softmax(s, lay, scale, out_dtype=torch.bfloat16, use_mask=False):
    """BlocksparseMaskedSoftmax<T,V> (blocksparse.h:649-722)."""
    return _host.masked_softmax(s, lay, scale, _DT[out_dtype], use_mask)


def bst_sgemm_xn(p, v, lay):
    """O = P.V over each block-row (bst_sgemm_xn with NN_OP, blocksparse.h:965-1014)."""
    return _host.bst_sgemm(p, v, lay, False)


def linear(x, w, bias=None, act=ACT_NONE, out=None):
    """out = act(x . w + bias) on the tensor cores: x [..., k], w [k, n] row-major, 16-bit; bias fp32 [n].
    The projections of the encoder layer with their bias add / GELU folded in
    (transformer_attention_optimize.cu:693-716, 755-763, 773-793)."""
    return _host.linear(x, w, bias, act, out, False)


def linear_nt(x, wt, bias=None, act=ACT_NONE, out=None):
    """out = act(x . wt^T + bias) with wt [n, k] row-major: the logits over the tied embedding table
    (transformer_inference_part.cpp:241)."""
    return _host.linear(x, wt, bias, act, out, True)


def embedding(table, ids, pos=None, scale=1.0):
    """out[b, l, :] = scale * table[ids[b, l], :] + pos[l, :] (embedding_lookup + tensor_add_matrix, embedding.h:5-12,
    ewops.h:276-282).  pos: of the table's type, L rows or more, of which the first L are read.  Returns (out, number of ids that were
    outside the table)."""
    return _host.embedding(table, ids, pos, scale)


def embedding_grad(dout, ids, vocab, scale=1.0, positions=False, dtype=torch.float32, out=None):
    """The gradients of embedding's tables from dout [B, L, hidden] and the same ids: dtable [vocab, hidden], scale times the sum of
    dout over the tokens of each id, and with positions dpos [L, hidden], its sum over the batch.  dtype: fp32 or dout's type (sums
    are fp32 either way, in a fixed order).  out: tensors (dtable, or with positions the pair) that the gradients are added to, such
    as a tied table's from the logits; None: new ones, zeros where an id does not occur.  Ids outside [0, vocab) have no row and are
    counted.  Returns (dtable, dpos or None, that count)."""
    return _host.embedding_grad(dout, ids, vocab, scale, positions, _DT[dtype], out)


def csr_from_layout(lay, head=0):
    """(rowptr, colidx): the element pattern of one head of a BlockLayout as CSR (every element of every kept block)."""
    bs, nb = lay.block_size, lay.nb
    dev = lay.layout.device
    rowptr = torch.empty(nb * bs + 1, dtype=torch.int32, device=dev)
    colidx = torch.empty(lay.blocks * bs * bs, dtype=torch.int32, device=dev)
    _check(lib.sfb_csr_from_layout(_stream(), _p(lay.layout[head]), nb, bs, _p(rowptr), _p(colidx)))
    return rowptr, colidx


def csr_attention(q, k, v, rowptr, colidx, scale):
    """Element-sparse attention over one CSR pattern shared by every (batch, head) (the reference's csr_* prototype,
    cuda_kernels.h:976-1075).  Returns (o, number of column indices that were outside the sequence)."""
    return _host.csr_attention(q, k, v, rowptr, colidx, scale)


def bst_sgemm_tn(a, b, lay):
    """C = A^T.B over each block column (bst_sgemm_xn with TN_OP, blocksparse.h:1005-1010): dV = P^T.dO and
    dK = dS^T.Q of the backward pass (transformer_attention_optimize.cu:924,954)."""
    return _host.bst_sgemm(a, b, lay, True)


def masked_softmax_grad(dy, y, lay, scale):
    """dx = (dy - sum_row(dy*y)) * y * scale (BlocksparseMaskedSoftmaxGrad<T,V>, blocksparse.h:1164-1227)."""
    return _host.masked_softmax_grad(dy, y, lay, scale)


def rowdot(a, b):
    """sum over the last dimension of a * b, fp32: delta = rowdot(dO, O) for the fused softmax gradient."""
    return _host.rowdot(a, b)


def fused_sddmm_softmax_grad(do, v, p, delta, lay, scale):
    """dS = P * (dO.V^T - delta) * scale in one launch (16-bit operands, 64x64 blocks, 64-wide heads)."""
    return _host.fused_sddmm_softmax_grad(do, v, p, delta, lay, scale)


def attention_backward_fused(q, k, v, p, o, do, lay, scale):
    """The backward with the dP / dS pair fused: dV = P^T.dO, dS = P*(dO.V^T - rowdot(dO, O))*scale, dK = dS^T.Q, dQ = dS.K.
    16-bit operands; o is the forward output.  Returns (dq, dk, dv)."""
    return _host.attention_backward_fused(do, q, k, v, p, o, lay, scale)


def attention_backward(q, k, v, p, do, lay, scale, s_dtype=torch.bfloat16):
    """The reference's backward sequence (transformer_attention_optimize.cu:924-964) from the saved probabilities:
    dV = P^T.dO, dP = dO.V^T, dS = softmax_grad(dP, P), dK = dS^T.Q, dQ = dS.K.  Returns (dq, dk, dv)."""
    return _host.attention_backward(do, q, k, v, p, lay, scale, _DT[s_dtype])


def fused_sddmm_softmax(q, k, lay, scale, out_dtype=torch.float32, use_mask=False):
    """P = softmax(scale * Q.K^T) in one launch (fusion_attention1/2/_full/_local/2_64,
    fusion_blocksparse.h:400,1212,1636,2030,2456)."""
    return _host.fused_sddmm_softmax(q, k, lay, scale, _DT[out_dtype], use_mask)


def fused_attention(q, k, v, lay, scale=None, use_mask=False, out=None):
    """O = softmax(scale * Q.K^T on the kept blocks).V in one launch (fusion_attention,
    fusion_blocksparse.h:2990-3050)."""
    return _host.fused_attention(q, k, v, lay, scale, use_mask, out)


def fused_attention_slice(q, k, v, lay, scale=None, use_mask=False, out=None):
    """fused_attention on views that select some heads (and batch elements) of wider [B, L, H_total, d] tensors, in
    place (sfb_fused_attention_slice): what one rank of a multi-GPU run calls on its share of the (batch, head) pairs."""
    return _host.fused_attention_slice(q, k, v, lay, scale, use_mask, out)


def fused_attention_stats(q, k, v, lay, scale=None, use_mask=False, out=None):
    """fused_attention for a training step: returns (o, lse), lse [B, H, L] the natural log of each row's sum of exp(scale * score) (fp32;
    -inf where a row keeps nothing), which is all that attention_backward_recompute needs of the probabilities.  q, k, v (and out)
    may be views that select some heads of wider [B, L, H_total, d] tensors, as in fused_attention_slice."""
    return _host.fused_attention_stats(q, k, v, lay, scale, use_mask, out)


def attention_backward_recompute(q, k, v, o, do, lse, lay, scale=None, use_mask=False, out=None):
    """The gradients (dq, dk, dv) of fused_attention_stats' output, with the probabilities made again from lse: nothing of the size
    of the scores is kept from one call to the other.  16-bit operands with blocks and heads of 64, all 16-byte aligned, have nothing of that size
    during the call either, as long as the layout has at most 256 block-rows or no row and column of more than 128 blocks.  Other calls go a slower
    way, by way of P and dS of some heads at a time in memory that torch's allocator has back after the call: up to 512 MB, or one head's where that
    is more (4 bytes per kept score, fp32 12: 2 GB for 16-bit causal heads of 32768 positions).  Any type, block and head size of the forward call; scale and use_mask as there.  q, k, v share a pitch, o and do
    have their own; out: three views to write to, of one pitch (such as the three parts of a packed [B, L, 3, H, d] gradient).  The same
    inputs give the same bits.  With 16-bit operands P and dS are rounded to their type as operands of the products.  The layout's tables
    by columns are built on first use (lay.tn_lut), which reads a number back: once before a call is captured in a graph."""
    return _host.attention_backward_recompute(q, k, v, o, do, lse, lay, scale, use_mask, out)


def grad_norm(grads, scale=1.0):
    """scale times the 2-norm over all elements of a list of tensors (fp32, bf16 and fp16 together; any dense layout), as a tensor of
    one fp32 element on their device.  The squares are summed in fp64, in a fixed order."""
    return _host.clip_grad_norm(grads, float("inf"), scale, None, False)


def clip_grad_norm(grads, max_norm, scale=1.0, out=None):
    """Multiplies every gradient by scale * min(1, max_norm / (norm + 1e-6)), norm = grad_norm(grads, scale): in place, or into the
    tensors of out (of the gradients' types or fp32: gradients of a scaled loss go, unscaled and clipped, into master gradients).
    Returns the norm; where it is infinite or NaN nothing is written.  Nothing is read back: the call can be captured in a graph."""
    return _host.clip_grad_norm(grads, max_norm, scale, out, True)


def bias_residual_layernorm(x, bias, resid, gain, beta, want_sum=False, out=None):
    """LayerNorm(resid + (x + bias)) (tensor_add_vector_gpu + tensor_add_tensor_gpu + layernorm_gpu,
    cuda_kernels.h:459,449,334).  Returns (out, sum or None, mean, rstd); out may be x or resid."""
    return _host.bias_residual_layernorm(x, bias, resid, gain, beta, want_sum, out)


def bias_gelu(x, bias, out=None):
    """(x + bias) * sigmoid(1.702 (x + bias)) (tensor_add_vector_gpu_2048 + gelu_gpu_v2, cuda_kernels.h:471,561)."""
    return _host.bias_gelu(x, bias, out)


def token_logprobs(logits, targets=None, vocab=None, scale=1.0, entropy=False, top_k=0):
    """Log probabilities of given tokens under softmax(scale * logits), with entropy and the top_k (at most 128) most probable
    tokens, in one pass over the logits: what linear_nt's result is scored by.

    logits [..., width] (fp32, bf16 or fp16; rows contiguous and at one pitch), targets int32 [...] or None.  vocab: how many
    columns are tokens (the rest is padding, as a table padded to a multiple of 16 leaves it).  Returns (logp, stats, entropy,
    top_logp, top_ids, missed), fp32 and int32, None for what was not asked for: stats [..., 2] holds each row's largest logit m
    and log sum exp(scale (x - m)), which the gradient needs.  Alternatives are in descending order, equal ones by ascending index; tokens at
    -inf are none (id -1, -inf).  A target outside [0, vocab) gives 0 and is counted in missed; such rows are not
    read (stats 0) unless entropy or alternatives are asked for.  To score each token by the logits before it, shift the targets and give
    each sequence's last row the target -1: logits[:, :-1] has no single pitch.

    The results of a call that has at most 64 KB of them, here and in the forward calls below, are views of one allocation: keeping
    (or saving) one keeps them all; clone() what is kept for long."""
    return _host.token_logprobs(logits, targets, vocab, scale, entropy, top_k)


def token_logprobs_grad(logits, targets, stats, dlogp, entropy=None, dentropy=None, vocab=None, scale=1.0, out=None):
    """The gradient of token_logprobs' logp and entropy with respect to the logits (in their type and layout; out may be logits):
    scale * (dlogp * (onehot - p) - dentropy * p * (log p + entropy)).  dlogp and dentropy are fp32 [...]; columns from vocab on
    get 0.  The alternatives' log probabilities have no gradient.  An out whose rows start elsewhere in
    their 16 bytes than the logits' do (a fresh one for logits[1:] of an odd width) is written element by element, which takes up to
    four times as long in 16 bits."""
    return _host.token_logprobs_grad(logits, targets, stats, dlogp, entropy, dentropy, vocab, scale, out)


def distill_topk(logits, ids, teacher, vocab=None, scale=1.0, tail=False):
    """KL divergence of the student's softmax(scale * logits) from a teacher's list of at most 128 tokens: ids int32 [..., k] and
    teacher fp32 [..., k], their log probabilities at the temperature (token_logprobs(teacher_logits, scale=scale, top_k=k)).
    The list is renormalised, or with tail=True what it leaves is one more class beside what the student leaves to unlisted
    tokens (left out of loss and gradient where all of those are at -inf).  Ids outside [0, vocab) are no entries (lists of uneven
    length) and are counted.  Returns (loss [...], stats [..., 2] or with tail [..., 3], missed).  The loss has no factor for the
    temperature."""
    return _host.distill_topk(logits, ids, teacher, vocab, scale, tail)


def distill_topk_grad(logits, ids, teacher, stats, dloss, vocab=None, scale=1.0, tail=False, targets=None, token_stats=None, dlogp=None,
                      out=None):
    """The gradient of distill_topk's loss with respect to the student's logits (out may be logits).  With targets, token_stats and dlogp
    (token_logprobs' stats at scale 1) the hard label's gradient dlogp * (onehot - softmax(logits)) is added in the same pass."""
    return _host.distill_topk_grad(logits, ids, teacher, stats, dloss, vocab, scale, tail, targets, token_stats, dlogp, out)


def linear_logprobs(x, table, targets, bias=None, vocab=None, scale=1.0, entropy=False):
    """token_logprobs(linear_nt(x, table, bias), targets) without the logits: scores of given tokens straight from hidden states
    x [..., k] over the (tied) table [n, k], 16-bit, k a multiple of 8.  Only the first vocab rows of the table are tokens (None: all;
    any number).  The logits are the tensor cores' fp32 sums, neither rounded nor stored: they drop what their additions
    shift out, 7e-7 of their norm from 64 bits at k = 768 and 2e-6 at 2048 (a plain fp32 product: 2 to 5e-7); for up to 128 rows and k
    above 512, 5e-7.  There is no gradient; training goes through linear_nt's logits.  Returns (logp, stats, entropy or None, missed) as token_logprobs does."""
    return _host.linear_logprobs(x, table, targets, bias, vocab, scale, entropy)


def encoder_layer_tensor(x2d, w, lay, heads, ln_order, scale):
    """One encoder layer on x2d [m, hidden] with every projection on this library's kernels (encoder.py's order)."""
    return _host.encoder_layer(x2d, w, lay, heads, ln_order == "pre", scale)


class HostPipeline:
    """Fused attention on operands that live in pinned HOST memory: the batch is cut into chunks and the
    host->device copies, the kernel and the device->host copy of consecutive chunks overlap on three streams
    (PCIe is full duplex, and the kernel is much shorter than either copy).  Device staging buffers are
    allocated once, here; a call allocates nothing."""

    def __init__(self, shape, dtype, lay, chunks=None, device="cuda"):
        B = shape[0]
        self.chunks = chunks or B
        assert B % self.chunks == 0
        self.lay = lay
        self.q, self.k, self.v, self.o = (torch.empty(shape, dtype=dtype, device=device) for _ in range(4))
        self.s_in, self.s_run, self.s_out = (torch.cuda.Stream(device=device) for _ in range(3))
        self.ev_in = [torch.cuda.Event() for _ in range(self.chunks)]
        self.ev_run = [torch.cuda.Event() for _ in range(self.chunks)]

    def __call__(self, hq, hk, hv, ho, scale):
        B = hq.shape[0]
        per = B // self.chunks
        cur = torch.cuda.current_stream()
        start = torch.cuda.Event()
        start.record(cur)
        for s in (self.s_in, self.s_run, self.s_out):
            s.wait_event(start)
        for c in range(self.chunks):
            sl = slice(c * per, (c + 1) * per)
            with torch.cuda.stream(self.s_in):
                self.q[sl].copy_(hq[sl], non_blocking=True)
                self.k[sl].copy_(hk[sl], non_blocking=True)
                self.v[sl].copy_(hv[sl], non_blocking=True)
                self.ev_in[c].record(self.s_in)
            with torch.cuda.stream(self.s_run):
                self.s_run.wait_event(self.ev_in[c])
                fused_attention(self.q[sl], self.k[sl], self.v[sl], self.lay, scale, out=self.o[sl])
                self.ev_run[c].record(self.s_run)
            with torch.cuda.stream(self.s_out):
                self.s_out.wait_event(self.ev_run[c])
                ho[sl].copy_(self.o[sl], non_blocking=True)
        done = torch.cuda.Event()
        done.record(self.s_out)
        cur.wait_event(done)
        return ho
