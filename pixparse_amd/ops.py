"""Tensor-level wrappers over the C-ABI (pixparse_amd.hip).  PyTorch is only the owner of device
memory and streams here: every function takes torch tensors, passes raw pointers + the current
HIP stream, and returns nothing that was computed by torch."""
import functools
from typing import Optional

import torch

from . import hip
from .hip import NT, NN, TN, EPI_BF16, EPI_BF16_GELU, EPI_BF16_DGELU, EPI_F32_RESID, EPI_F32, EPI_F32_ACC  # noqa: F401

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
_FUSE_DBIAS = __import__('os').environ.get('PIXPARSE_AMD_FUSE_DBIAS', '1') != '0'     # A/B switch: bias gradients from the weight-gradient GEMM (default) or a pass of their own
VOCAB_PAD = 128   # logits row stride / embedding rows are padded to a multiple of this
K_PAD = 64        # contraction dims of NT/NN GEMMs are padded to a multiple of this when needed


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def round_up(x: int, m: int) -> int:
    return (x + m - 1) // m * m


def _chk(t: torch.Tensor, dtype, name: str):
    if t.dtype != dtype or not t.is_cuda:
        raise TypeError(f'{name}: expected a cuda {dtype} tensor, got {t.dtype} on {t.device}')


def gemm(layout: int, epi: int, M: int, N: int, K: int, A: torch.Tensor, lda: int, B: torch.Tensor, ldb: int,
         C: torch.Tensor, ldc: int, bias: Optional[torch.Tensor] = None, aux: Optional[torch.Tensor] = None,
         ldaux: int = 0, resid: Optional[torch.Tensor] = None, ldr: int = 0, colscale: float = 1.0, colscale_cols: int = 0) -> None:
    _chk(A, BF16, 'gemm A')
    _chk(B, BF16, 'gemm B')
    ws = None
    _gemm_env()
    wsb = hip.query('crl_gemm_ws_bytes', layout, epi, M, N, K)   # wgrad split-K slabs, or the split remainder rows of a forward / dgrad GEMM
    if wsb:
        ws = _gemm_scratch.get(wsb, A.device)
    hip.call('crl_gemm_bf16', layout, epi, M, N, K, _p(A), lda, _p(B), ldb, _p(bias), _p(C), ldc, _p(aux), ldaux,
             _p(resid), ldr, float(colscale), int(colscale_cols), _p(ws), wsb, _stream())


_gemm_env_applied = False


def _gemm_env():
    """A/B switches of the GEMM dispatch, read once: PIXPARSE_AMD_GEMM_BIG=0|1|2 (crl_gemm_set_big_kernel: 8-wave / 4-wave / per launch),
    PIXPARSE_AMD_GEMM_OVERLAP=0|1 (crl_gemm_set_overlap)"""
    global _gemm_env_applied
    if _gemm_env_applied:
        return
    _gemm_env_applied = True
    import os
    for env, fn in (('PIXPARSE_AMD_GEMM_BIG', 'crl_gemm_set_big_kernel'), ('PIXPARSE_AMD_GEMM_OVERLAP', 'crl_gemm_set_overlap')):
        if os.environ.get(env):
            hip.call(fn, int(os.environ[env]))


_calibrated = {}


def gemm_calibrate(device, force: bool = False):
    """one-off per process and device: refit the wave-quantisation cost model of the persistent GEMMs to what THIS device sustains
    (crl_gemm_calibrate; synchronises).  OPT-IN since round 5 (PIXPARSE_AMD_GEMM_CALIBRATE=1, or force=True): the fitted constants decide
    where the wave-quantisation cut falls, i.e. which rows take the split-contraction path with its different summation order, so a default-on
    timing fit made the bits of every large GEMM depend on measurement noise (run to run, rank to rank, across a resume) for no
    measured gain (244.3 vs 244.0 ms).  Returns (a_us, b_us, calibrated)."""
    import ctypes
    import os
    key = str(device)
    # (two ranks sharing one device -- CRL_DEBUG_SHARED_GPU, a validation aid -- would time each other's launches: built-in constants there)
    if (force or (key not in _calibrated and os.environ.get('PIXPARSE_AMD_GEMM_CALIBRATE', '0') == '1')) and os.environ.get('CRL_DEBUG_SHARED_GPU', '0') != '1':
        nbytes = hip.query('crl_gemm_calibrate_ws_bytes')
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)      # its own buffer: released again right away
        rc = hip.load().crl_gemm_calibrate(_p(ws), nbytes, _stream())
        if rc < 0:
            raise hip.HipLibraryError(f'crl_gemm_calibrate failed ({rc}): {hip.last_error()}')
        del ws
        _calibrated[key] = rc
    a, b, c = ctypes.c_float(), ctypes.c_float(), ctypes.c_int()
    hip.call('crl_gemm_model', ctypes.addressof(a), ctypes.addressof(b), ctypes.addressof(c))
    return a.value, b.value, bool(c.value)


def linear_fwd(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor, epi: int = EPI_BF16,
               aux: Optional[torch.Tensor] = None, resid: Optional[torch.Tensor] = None, n: Optional[int] = None,
               colscale: float = 1.0, colscale_cols: int = 0) -> None:
    """out[M, N] = x[M, K] @ w[N, K]^T (+bias) with the epilogue; x, w bf16 row-major 2-D (may be row-strided).
    colscale / colscale_cols: the first colscale_cols output columns are multiplied by colscale before the bf16 rounding (q of q|k|v)."""
    M, K = x.shape
    N = n if n is not None else w.shape[0]
    gemm(NT, epi, M, N, K, x, x.stride(0), w, w.stride(0), out, out.stride(0), bias, aux,
         aux.stride(0) if aux is not None else 0, resid, resid.stride(0) if resid is not None else 0, colscale, colscale_cols)


SKINNY_MAX_ROWS = 16


def linear_skinny(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor, epi: int = EPI_BF16,
                  resid: Optional[torch.Tensor] = None, n: Optional[int] = None, out_row: Optional[torch.Tensor] = None,
                  out_row_stride: int = 0) -> None:
    """decode-time linear_fwd for M <= 16 rows (crl_linear_skinny_bf16): every weight byte read once, no tiles.
    out_row (device int32 scalar): the output is shifted by out_row * out_row_stride elements (KV-cache row of the step)."""
    M, K = x.shape
    N = n if n is not None else w.shape[0]
    hip.call('crl_linear_skinny_bf16', epi, M, N, K, _p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(out), out.stride(0),
             _p(resid), resid.stride(0) if resid is not None else 0, _p(out_row), int(out_row_stride), _stream())


def linear_skinny_ln(x32: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, h32: Optional[torch.Tensor], w: torch.Tensor,
                     bias: Optional[torch.Tensor], out: torch.Tensor, epi: int = EPI_BF16, n: Optional[int] = None,
                     out_row: Optional[torch.Tensor] = None, out_row_stride: int = 0) -> None:
    """out = epilogue(bf16(LayerNorm(x32)) @ w^T + bias) for M <= 16 rows, h32 (optional) = the fp32 LayerNorm output
    (crl_linear_skinny_ln_bf16: the LayerNorm in front of a decode-step projection without a launch of its own)"""
    M, K = x32.shape
    N = n if n is not None else w.shape[0]
    hip.call('crl_linear_skinny_ln_bf16', epi, M, N, K, _p(x32), x32.stride(0), _p(gamma), _p(beta), float(eps), _p(h32),
             h32.stride(0) if h32 is not None else 0, _p(w), w.stride(0), _p(bias), _p(out), out.stride(0), _p(out_row), int(out_row_stride), _stream())


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, out: torch.Tensor, epi: int = EPI_BF16,
                 aux: Optional[torch.Tensor] = None, k: Optional[int] = None) -> None:
    """out[M, Kin] = dy[M, N] @ w[N, Kin]; contraction over N (= dy.shape[1])."""
    M, N = dy.shape
    Kin = k if k is not None else w.shape[1]
    gemm(NN, epi, M, Kin, N, dy, dy.stride(0), w, w.stride(0), out, out.stride(0), None, aux,
         aux.stride(0) if aux is not None else 0)


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor, accumulate: bool = True,
                 n: Optional[int] = None, k: Optional[int] = None, dbias: Optional[torch.Tensor] = None, dbias_accumulate: bool = True) -> None:
    """dw[N, Kin] (+)= dy[M, N]^T @ x[M, Kin]  (fp32 output straight into the grad arena).
    dbias (optional, fp32 [N]): the bias gradient dbias[n] (+)= sum_m dy[m, n] from the SAME call -- the 4-wave weight-gradient kernel sums the
    columns of its A operand on the matrix pipe while it streams them (crl_gemm_bf16, CRL_TN with aux); any other kernel: the column-sum pass."""
    M = dy.shape[0]
    N = n if n is not None else dy.shape[1]
    Kin = k if k is not None else x.shape[1]
    if dbias is not None:
        _chk(dbias, F32, 'linear_wgrad dbias')
        if not _FUSE_DBIAS:       # A/B switch (PIXPARSE_AMD_FUSE_DBIAS=0): the separate column-sum pass of rounds 1-5
            gemm(TN, EPI_F32_ACC if accumulate else EPI_F32, N, Kin, M, dy, dy.stride(0), x, x.stride(0), dw, dw.stride(0))
            colsum(dy, dbias, dbias_accumulate, n=n)
            return
    gemm(TN, EPI_F32_ACC if accumulate else EPI_F32, N, Kin, M, dy, dy.stride(0), x, x.stride(0), dw, dw.stride(0),
         aux=dbias, ldaux=1 if (dbias is not None and dbias_accumulate) else 0)


class Scratch:
    """lazily grown device scratch shared by the reductions (never read across calls).  Once a hipGraph has been captured
    (freeze_scratch()) a buffer that has to grow is RETIRED, not freed: the graph's launches keep writing their slabs / partials into
    the address they were captured with, which stays owned by this object instead of going back to the caching allocator where other
    tensors would be handed the same memory; from then on it grows by at least half its size."""
    frozen = False

    def __init__(self):
        self.buf = None
        self.retired = []

    def get(self, nbytes: int, device) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < nbytes or self.buf.device != device:
            want = max(nbytes, 1 << 20)
            if Scratch.frozen and self.buf is not None:
                self.retired.append(self.buf)
                # a retired buffer is never released: grow geometrically so that a rising sequence of requests (eval / generation shapes after a
                # graphed training run) retires at most ~2 x the final size in all, not one buffer per request
                if self.buf.device == device:
                    want = max(want, self.buf.numel() + self.buf.numel() // 2)
            self.buf = torch.empty(want, dtype=torch.uint8, device=device)
            import os
            if os.environ.get('PIXPARSE_AMD_POISON', '0') == '1':    # debug aid (see layers/engines.py Buffers)
                self.buf.fill_(255)
        return self.buf


def freeze_scratch() -> None:
    """call before capturing launches into a hipGraph: from now on scratch buffers are never released (see Scratch)"""
    Scratch.frozen = True


_scratch = Scratch()
_gemm_scratch = Scratch()
_attn_scratch = Scratch()


def colsum(x: torch.Tensor, out: torch.Tensor, accumulate: bool = True, n: Optional[int] = None) -> None:
    M = x.shape[0]
    N = n if n is not None else x.shape[1]
    ws = _scratch.get(hip.query('crl_colsum_ws_bytes', N), x.device)
    hip.call('crl_colsum_bf16', _p(x), M, N, x.stride(0), _p(out), int(accumulate), _p(ws), _stream())


def layernorm_fwd(x, gamma, beta, eps, y_f32, y_bf16, mean, rstd) -> None:
    M, D = x.shape
    _chk(x, F32, 'layernorm x')
    hip.call('crl_layernorm_fwd', _p(x), _p(gamma), _p(beta), float(eps), M, D, _p(y_f32), _p(y_bf16), _p(mean), _p(rstd),
             _stream())


def layernorm_bwd(dy_f32, dy_bf16, x, gamma, mean, rstd, dx_f32, dx_accumulate, dx_bf16, dgamma, dbeta,
                  acc_wgrad: bool = True, dx_colsum: Optional[torch.Tensor] = None) -> None:
    """dx_colsum [D] (+)= column sums of the bf16 gradient written to dx_bf16 (the bias gradient of the Linear it feeds)"""
    M, D = x.shape
    assert dx_colsum is None or dx_bf16 is not None
    ws = _scratch.get(hip.query('crl_layernorm_bwd_ws_bytes', D), x.device)
    hip.call('crl_layernorm_bwd', _p(dy_f32), _p(dy_bf16), _p(x), _p(gamma), _p(mean), _p(rstd), M, D, _p(dx_f32),
             int(dx_accumulate), _p(dx_bf16), _p(dgamma), _p(dbeta), _p(dx_colsum), int(acc_wgrad), _p(ws), _stream())


HEAD_DIM = 64   # the attention kernels index head h at channel h * 64


def _chk_heads(heads: int, *tensors) -> None:
    for t in tensors:
        if t.shape[-1] != heads * HEAD_DIM:
            raise ValueError(f'attention kernels are built for head_dim {HEAD_DIM}: got {t.shape[-1]} channels for {heads} heads '
                             f'(head_dim {t.shape[-1] / max(heads, 1):g})')


def _bs_rs(t: torch.Tensor):
    """(batch stride, row stride) in elements of a [B, N, H*64-ish] view whose last dim is contiguous."""
    assert t.dim() == 3 and t.stride(2) == 1, 'attention operands are [B, N, H*64] views with contiguous channels'
    return t.stride(0), t.stride(1)


def _drop_args(drop, site):
    """(p, seed, step, site) of an attention-probability dropout call; drop: DropSpec-like with .p_attn (None / 0 = off)"""
    if drop is None or not getattr(drop, 'p_attn', 0.0):
        return 0.0, 0, 0, 0
    return float(drop.p_attn), drop.seed, drop.step, int(site)


LOG2E = 1.4426950408889634


_attn_fwd_env_applied = False


def attn_fwd(q, k, v, o, lse, heads: int, scale: float, causal: bool, drop=None, site: int = 0, q_prescaled: bool = False) -> None:
    """q [B,Nq,H*64], k/v [B,Nk,H*64] (strided views allowed), o like q, lse [B,H,Nq] f32.
    drop (DropSpec with p_attn > 0) + site: dropout of the attention probabilities (the backward call must pass the same pair).
    q_prescaled: q already carries scale * log2(e) (linear_fwd(..., colscale=scale * LOG2E, colscale_cols=D)): the faster forward kernel."""
    global _attn_fwd_env_applied
    if not _attn_fwd_env_applied:      # A/B switch: PIXPARSE_AMD_ATTN_FWD_MODE=1 the compiler-scheduled kernels, 3 / 4 the stream at one / two workgroups per CU
        import os
        _attn_fwd_env_applied = True
        if os.environ.get('PIXPARSE_AMD_ATTN_FWD_MODE'):
            hip.call('crl_attn_fwd_set_mode', int(os.environ['PIXPARSE_AMD_ATTN_FWD_MODE']))
        if os.environ.get('PIXPARSE_AMD_ATTN_FWD_PERSIST'):     # 0: one workgroup per query block instead of the persistent launch
            hip.call('crl_attn_fwd_set_persistent', int(os.environ['PIXPARSE_AMD_ATTN_FWD_PERSIST']))
    B, Nq, _ = q.shape
    Nk = k.shape[1]
    _chk_heads(heads, q, k, v, o)
    hip.call('crl_attn_fwd', _p(q), *_bs_rs(q), _p(k), *_bs_rs(k), _p(v), *_bs_rs(v), _p(o), *_bs_rs(o), _p(lse),
             B, heads, Nq, Nk, float(scale), int(causal), int(q_prescaled), *_drop_args(drop, site), _stream())


def attn_dropout_mask(B: int, H: int, Nq: int, Nk: int, drop, site: int, device) -> torch.Tensor:
    """the keep mask [B, H, Nq, Nk] (uint8) the attention kernels regenerate for (drop, site)"""
    keep = torch.empty(B, H, Nq, Nk, dtype=torch.uint8, device=device)
    p, seed, step, st = _drop_args(drop, site)
    hip.call('crl_attn_dropout_mask', _p(keep), B, H, Nq, Nk, p, seed, step, st, _stream())
    return keep


def attn_decode(q, k, v, o, heads: int, scale: float, nk_minus1: Optional[torch.Tensor] = None,
                q_row: Optional[torch.Tensor] = None, q_row_stride: int = 0) -> None:
    """single-query attention over a KV cache: q, o [B, H*64] (row-strided), k / v [B, Nk, H*64] strided views.
    nk_minus1 (device int32 scalar): only the first nk_minus1 + 1 keys are valid (k.shape[1] is the capacity);
    q_row: q is taken q_row * q_row_stride elements further (the step's cache row)."""
    B = q.shape[0]
    Nk = k.shape[1]
    assert q.dim() == 2 and q.stride(1) == 1 and o.stride(1) == 1
    _chk_heads(heads, q, k, v, o)
    nbytes = hip.query('crl_attn_decode_ws_bytes', B, heads, Nk)
    ws = _scratch.get(nbytes, q.device)
    hip.call('crl_attn_decode', _p(q), q.stride(0), _p(k), *_bs_rs(k), _p(v), *_bs_rs(v), _p(o), o.stride(0), B, heads, Nk,
             float(scale), _p(nk_minus1), _p(q_row), int(q_row_stride), _p(ws), nbytes, _stream())


# ------------------------------------------------------------------------------------------- a key-value cache in pages
# A call on a few rows takes the GPU 5 us, so the checks of the operators below are one expression over attributes that are read once; a call
# that does not pass it goes to the function behind `refuse`, which finds the reason and raises it.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, '_cuda_getCurrentRawStream') else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run_on(index: int, name: str, *args) -> None:
    """hip.call(name, *args, the current stream of device `index`), with that device the current one"""
    if index == torch.cuda.current_device():
        rc = getattr(hip.load(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(hip.load(), name)(*args, _raw_stream(index))
    if rc != 0:
        raise hip.HipLibraryError(f'{name} failed ({rc}): {hip.last_error()}')


def _want(t: Optional[torch.Tensor], name: str, dtype, *shape) -> None:
    """raises unless the operand (None: left out) has this dtype, this shape (None: any size) and a contiguous last dimension"""
    if t is None:
        return
    if t.dtype != dtype:
        raise TypeError(f'{name}: expected {dtype}, got {t.dtype}')
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise ValueError(f'{name}: expected shape {tuple("any" if w is None else w for w in shape)}, got {tuple(t.shape)}')
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')


def _want_rows(t: Optional[torch.Tensor], name: str, width: int) -> None:
    """raises where the rows of an output overlap"""
    if t is not None and any(n > 1 and s < width for n, s in zip(t.shape[:-1], t.stride()[:-1])):
        raise ValueError(f'{name}: rows overlap (strides {t.stride()})')


def _want_one_device(*tensors) -> None:
    devs = {t.device for t in tensors if t is not None}
    if len(devs) != 1 or next(iter(devs)).type != 'cuda':
        raise TypeError(f'expected tensors of one cuda device, got {sorted(str(d) for d in devs)}')


def _refuse_pool(k_pages, v_pages, page_table, weights, B: int) -> int:
    """pool [pages, page_size, kv_heads, 64] (strided views, k and v alike), page table [B, n] int32, weights [B, kv_heads, >= positions]"""
    _want(k_pages, 'k_pages', BF16, None, None, None, HEAD_DIM)
    _want(v_pages, 'v_pages', BF16, *k_pages.shape)
    _want(page_table, 'page_table', torch.int32, B, None)
    if k_pages.stride() != v_pages.stride():
        raise ValueError(f'k_pages and v_pages must have the same strides, got {k_pages.stride()} and {v_pages.stride()}')
    kv_heads, positions = k_pages.shape[2], k_pages.shape[1] * page_table.shape[1]
    if weights is not None:
        _want(weights, 'weights', F32, B, kv_heads, None)
        if weights.shape[2] < positions:
            raise ValueError(f'weights: {weights.shape[2]} positions, the page table covers {positions}')
        _want_rows(weights, 'weights', positions)
    return kv_heads


def _pool_ok(k_pages, v_pages, ks, sh, page_table, ts, tn, weights, ws, B: int, index: int) -> bool:
    return (len(sh) == 4 and sh[3] == HEAD_DIM and ks[3] == 1 and v_pages.shape == sh and v_pages.stride() == ks and k_pages.dtype is BF16
            and v_pages.dtype is BF16 and len(tn) == 2 and tn[0] == B and ts[1] == 1 and page_table.dtype is torch.int32
            and k_pages.get_device() == index == v_pages.get_device() == page_table.get_device()
            and (weights is None or (weights.dtype is F32 and len(ws) == 3 and ws[2] == 1 and weights.get_device() == index
                                     and weights.shape[:2] == (B, sh[2]) and weights.shape[2] >= sh[1] * tn[1] <= min(ws[0], ws[1]))))


def _vectors_ok(B: int, index: int, *vectors) -> bool:
    return all(t.dtype is torch.int32 and t.shape == (B,) and t.is_contiguous() and t.get_device() == index for t in vectors)


def _refuse(names, locals_, *checks):
    """runs the checks one after the other; what passes them all is on the wrong device"""
    for c in checks:
        c()
    _want_one_device(*(locals_[n] for n in names))
    raise ValueError('operands of this layout are not supported: ' + ', '.join(f'{n} {tuple(locals_[n].shape)} {locals_[n].stride()}'
                                                                                for n in names if locals_[n] is not None))


@functools.lru_cache(maxsize=4096)
def _paged_ws_bytes(B: int, heads: int, kv_heads: int, page_size: int, pages: int, weights: bool) -> int:
    return hip.query('crl_paged_attn_decode_ws_bytes', B, heads, kv_heads, page_size, pages, int(weights))


def paged_attn_decode(q, k_pages, v_pages, page_table, lengths, o, heads: int, scale: float, k_new: Optional[torch.Tensor] = None,
                      v_new: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None) -> None:
    """attn_decode over a cache in pages, every sequence at a length of its own: q, o [B, H*64] bf16 (row-strided), k_pages / v_pages
    [pages, page_size, kv_heads, 64] bf16 (strided, alike; H a multiple of kv_heads), page_table [B, n] and lengths [B] int32 on the device.
    Position p of sequence b is row p % page_size of page page_table[b, p // page_size].  A length of 0 gives zeros; a length outside the table
    or a page outside the pool gives NaN.
    k_new / v_new [B, kv_heads*64]: the rows of position lengths - 1, which the call also writes to their pages.
    weights [B, kv_heads, >= n * page_size] fp32: the attention weights are added to it (what cache_evict chooses by); the position of an
    appended row starts from 0."""
    qn, qs, os_, sh, ks, tn, ts = q.shape, q.stride(), o.stride(), k_pages.shape, k_pages.stride(), page_table.shape, page_table.stride()
    B, index = qn[0], q.get_device()
    ws = weights.stride() if weights is not None else (0, 0, 0)
    kns, vns = (k_new.stride(), v_new.stride()) if k_new is not None and v_new is not None else ((0, 1), (0, 1))
    if not (index >= 0 and len(qn) == 2 and qn[1] == heads * HEAD_DIM and o.shape == qn and qs[1] == 1 == os_[1] and os_[0] >= qn[1]
            and q.dtype is BF16 and o.dtype is BF16 and o.get_device() == index and (k_new is None) == (v_new is None)
            and _pool_ok(k_pages, v_pages, ks, sh, page_table, ts, tn, weights, ws, B, index) and heads > 0 and sh[2] > 0 and heads % sh[2] == 0
            and _vectors_ok(B, index, lengths)
            and (k_new is None or (k_new.dtype is BF16 and v_new.dtype is BF16 and k_new.shape == (B, sh[2] * HEAD_DIM) == v_new.shape
                                   and kns[1] == 1 == vns[1] and k_new.get_device() == index == v_new.get_device()))):
        _refuse_paged_attn(q, k_pages, v_pages, page_table, lengths, o, heads, k_new, v_new, weights)
    nbytes = _paged_ws_bytes(B, heads, sh[2], sh[1], tn[1], weights is not None)
    # a workspace of the call's own: of the current stream and, under capture, of the graph
    buf = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _run_on(index, 'crl_paged_attn_decode', q.data_ptr(), qs[0], k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], sh[0], sh[1],
            page_table.data_ptr(), ts[0], tn[1], lengths.data_ptr(), _p(k_new), kns[0], _p(v_new), vns[0], o.data_ptr(), os_[0], _p(weights),
            ws[0], ws[1], B, heads, sh[2], scale, _p(buf), nbytes)


def _refuse_paged_attn(q, k_pages, v_pages, page_table, lengths, o, heads, k_new, v_new, weights):
    def shapes():
        B = q.shape[0]
        kv_heads = _refuse_pool(k_pages, v_pages, page_table, weights, B)
        if heads <= 0 or kv_heads == 0 or heads % kv_heads:
            raise ValueError(f'{heads} query heads do not divide into {kv_heads} key-value heads')
        _chk_heads(heads, q, o)
        _want(q, 'q', BF16, B, heads * HEAD_DIM)
        _want(o, 'o', BF16, B, heads * HEAD_DIM)
        _want_rows(o, 'o', heads * HEAD_DIM)
        _want(lengths, 'lengths', torch.int32, B)
        if (k_new is None) != (v_new is None):
            raise ValueError('k_new and v_new go together')
        _want(k_new, 'k_new', BF16, B, kv_heads * HEAD_DIM)
        _want(v_new, 'v_new', BF16, B, kv_heads * HEAD_DIM)
        if not lengths.is_contiguous():
            raise ValueError('lengths must be contiguous')
    _refuse(('q', 'k_pages', 'v_pages', 'page_table', 'lengths', 'o', 'k_new', 'v_new', 'weights'), locals(), shapes)


def paged_append(k, v, k_pages, v_pages, page_table, starts, counts, weights: Optional[torch.Tensor] = None) -> None:
    """rows k / v [B, T, kv_heads*64] bf16 (strided views, e.g. of a q|k|v projection) -> positions starts[b] + t, t < counts[b] (int32 [B],
    device) of a cache in pages (see paged_attn_decode).  weights: set to 0 at those positions.  Rows outside the table or the pool are
    dropped."""
    kn, kst, vst, sh, ks, tn, ts = k.shape, k.stride(), v.stride(), k_pages.shape, k_pages.stride(), page_table.shape, page_table.stride()
    B, index = kn[0], k.get_device()
    ws = weights.stride() if weights is not None else (0, 0, 0)
    if not (index >= 0 and _pool_ok(k_pages, v_pages, ks, sh, page_table, ts, tn, weights, ws, B, index) and len(kn) == 3 and kn[1] > 0
            and kn[2] == sh[2] * HEAD_DIM and v.shape == kn and kst[2] == 1 == vst[2] and k.dtype is BF16 and v.dtype is BF16
            and v.get_device() == index and _vectors_ok(B, index, starts, counts)):
        _refuse_append(k, v, k_pages, v_pages, page_table, starts, counts, weights)
    _run_on(index, 'crl_paged_append', k.data_ptr(), kst[0], kst[1], v.data_ptr(), vst[0], vst[1], k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1],
            ks[2], sh[0], sh[1], page_table.data_ptr(), ts[0], tn[1], starts.data_ptr(), counts.data_ptr(), _p(weights), ws[0], ws[1], B, kn[1], sh[2])


def _refuse_append(k, v, k_pages, v_pages, page_table, starts, counts, weights):
    def shapes():
        B = k.shape[0]
        kv_heads = _refuse_pool(k_pages, v_pages, page_table, weights, B)
        _want(k, 'k', BF16, B, None, kv_heads * HEAD_DIM)
        _want(v, 'v', BF16, *k.shape)
        if k.shape[1] == 0:
            raise ValueError('k: no rows to append')
        for t, name in ((starts, 'starts'), (counts, 'counts')):
            _want(t, name, torch.int32, B)
            if not t.is_contiguous():
                raise ValueError(f'{name} must be contiguous')
    _refuse(('k', 'v', 'k_pages', 'v_pages', 'page_table', 'starts', 'counts', 'weights'), locals(), shapes)


def cache_evict(k_pages, v_pages, page_table, lengths, weights, budget: int, recent: int, new_lengths,
                kept: Optional[torch.Tensor] = None) -> None:
    """cuts every sequence of a cache in pages that is longer than `budget` down to it, per key-value head: the last `recent` positions and, of the
    others, those with the largest weights (weights [B, kv_heads, positions] fp32, as paged_attn_decode gathers them; equal ones: the lower
    position) move to positions 0 .. budget - 1, in order, in place, with their weights.  new_lengths [B] int32 (may be lengths itself)
    receives min(lengths, budget); kept [B, kv_heads, budget] int32 (optional) the positions that stayed, -1 behind the last.  The pages of
    a sequence must be its own.  A sequence with a length outside the table, or one to be cut with a page outside the pool, stays whole (kept: -1)."""
    tn, ts, sh, ks = page_table.shape, page_table.stride(), k_pages.shape, k_pages.stride()
    B, index = tn[0], k_pages.get_device()
    ws = weights.stride() if weights is not None else None
    if not (ws is not None and index >= 0 and _pool_ok(k_pages, v_pages, ks, sh, page_table, ts, tn, weights, ws, B, index)
            and _vectors_ok(B, index, lengths, new_lengths) and budget >= 1 and 0 <= recent <= budget
            and (kept is None or (kept.dtype is torch.int32 and kept.shape == (B, sh[2], budget) and kept.is_contiguous() and kept.get_device() == index))):
        _refuse_evict(k_pages, v_pages, page_table, lengths, weights, budget, recent, new_lengths, kept)
    if kept is None:                       # (what no sequence can reach needs no list)
        budget = min(budget, max(1, sh[1] * tn[1]))
        recent = min(recent, budget)
    nbytes = 4 * B * sh[2] * (1 if kept is not None else budget + 1)
    buf = torch.empty(nbytes, dtype=torch.uint8, device=k_pages.device)
    _run_on(index, 'crl_cache_evict', k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], sh[0], sh[1], page_table.data_ptr(), ts[0], tn[1],
            lengths.data_ptr(), weights.data_ptr(), ws[0], ws[1], B, sh[2], budget, recent, new_lengths.data_ptr(), _p(kept), buf.data_ptr(), nbytes)


def _refuse_evict(k_pages, v_pages, page_table, lengths, weights, budget, recent, new_lengths, kept):
    def shapes():
        B = page_table.shape[0]
        if weights is None:
            raise ValueError('weights: needed to choose by')
        kv_heads = _refuse_pool(k_pages, v_pages, page_table, weights, B)
        _want(lengths, 'lengths', torch.int32, B)
        _want(new_lengths, 'new_lengths', torch.int32, B)
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f'budget {budget}, recent {recent}: 0 <= recent <= budget, budget >= 1')
        _want(kept, 'kept', torch.int32, B, kv_heads, int(budget))
        if not lengths.is_contiguous() or not new_lengths.is_contiguous() or (kept is not None and not kept.is_contiguous()):
            raise ValueError('lengths, new_lengths and kept must be contiguous')
    _refuse(('k_pages', 'v_pages', 'page_table', 'lengths', 'weights', 'new_lengths', 'kept'), locals(), shapes)


def embed_decode(ids, tok, pos, out, step: torch.Tensor, pos_offset: int = 2) -> None:
    """generation: ids [B, 1] at position `step` (device int32 scalar) -> out f32 [B, D]"""
    hip.call('crl_embed_decode', _p(ids), _p(tok), _p(pos), _p(out), ids.shape[0], out.shape[1], pos_offset, tok.shape[0], _p(step),
             _stream())


def embed_decode_rows(ids, tok, pos, out, positions: torch.Tensor, pos_offset: int = 2) -> None:
    """generation of sequences at positions of their own: ids [B, 1] at positions [B] (device int32) -> out f32 [B, D]"""
    B, D = out.shape
    for t, name, dtype, shape in ((ids, 'ids', torch.int64, (B, 1)), (tok, 'tok', F32, (None, D)), (pos, 'pos', F32, (None, D)), (out, 'out', F32, (B, D)),
                                  (positions, 'positions', torch.int32, (B,))):
        _want(t, name, dtype, *shape)
        if not t.is_contiguous():
            raise ValueError(f'{name} must be contiguous')
    _want_one_device(ids, tok, pos, out, positions)
    _run_on(out.get_device(), 'crl_embed_decode_rows', ids.data_ptr(), tok.data_ptr(), pos.data_ptr(), out.data_ptr(), B, D, pos_offset, tok.shape[0],
            positions.data_ptr(), pos.shape[0])


_attn_mode_env_applied = False


def attn_bwd(q, k, v, o, d_o, lse, delta, dq, dk, dv, heads: int, scale: float, causal: bool, drop=None, site: int = 0,
             q_prescaled: bool = False) -> None:
    global _attn_mode_env_applied
    if not _attn_mode_env_applied:      # A/B switch: PIXPARSE_AMD_ATTN_BWD_MODE=1 forces the two-pass backward, 2 the single pass (crl_attn_bwd_set_mode)
        import os
        _attn_mode_env_applied = True
        if os.environ.get('PIXPARSE_AMD_ATTN_BWD_MODE'):
            hip.call('crl_attn_bwd_set_mode', int(os.environ['PIXPARSE_AMD_ATTN_BWD_MODE']))
        if os.environ.get('PIXPARSE_AMD_ATTN_BWD_QSPLIT'):  # query split of the single pass's remainder chains (crl_attn_bwd_set_qsplit; -1 = auto)
            hip.call('crl_attn_bwd_set_qsplit', int(os.environ['PIXPARSE_AMD_ATTN_BWD_QSPLIT']))
        if os.environ.get('PIXPARSE_AMD_ATTN_BWD_PERSIST'):  # 0: one workgroup per chain instead of the persistent ticket-pulling launch (crl_attn_bwd_set_persistent)
            hip.call('crl_attn_bwd_set_persistent', int(os.environ['PIXPARSE_AMD_ATTN_BWD_PERSIST']))
        if os.environ.get('PIXPARSE_AMD_ATTN_BWD_CHAIN'):   # key blocks per workgroup of the single pass (crl_attn_bwd_set_chain; 0 = auto)
            hip.call('crl_attn_bwd_set_chain', int(os.environ['PIXPARSE_AMD_ATTN_BWD_CHAIN']))
    B, Nq, _ = q.shape
    Nk = k.shape[1]
    _chk_heads(heads, q, k, v, o, d_o, dq, dk, dv)
    wsb = hip.query('crl_attn_bwd_ws_bytes', B, heads, Nq, Nk, int(causal))     # partial-dQ slabs of the single-pass form (0: two-pass)
    ws = _attn_scratch.get(wsb, q.device) if wsb else None
    hip.call('crl_attn_bwd', _p(q), *_bs_rs(q), _p(k), *_bs_rs(k), _p(v), *_bs_rs(v), _p(o), *_bs_rs(o),
             _p(d_o), *_bs_rs(d_o), _p(lse), _p(delta), _p(dq), *_bs_rs(dq), _p(dk), *_bs_rs(dk), _p(dv), *_bs_rs(dv),
             B, heads, Nq, Nk, float(scale), int(causal), int(q_prescaled), *_drop_args(drop, site), _p(ws), wsb, _stream())


def swin_attn_fwd(qkv, table, out, B, Hf, Wf, heads, w, shift, scale) -> None:
    hip.call('crl_swin_attn_fwd', _p(qkv), _p(table), _p(out), B, Hf, Wf, heads, w, shift, float(scale), _stream())


def swin_attn_bwd(qkv, table, d_out, dqkv, dtable, B, Hf, Wf, heads, w, shift, scale) -> None:
    hip.call('crl_swin_attn_bwd', _p(qkv), _p(table), _p(d_out), _p(dqkv), _p(dtable), B, Hf, Wf, heads, w, shift,
             float(scale), _stream())


def patch_merge_fwd(x, y, B, Hf, Wf, C) -> None:
    hip.call('crl_patch_merge_fwd', _p(x), _p(y), B, Hf, Wf, C, _stream())


def patch_merge_bwd(dy, dx, B, Hf, Wf, C) -> None:
    hip.call('crl_patch_merge_bwd', _p(dy), _p(dx), B, Hf, Wf, C, _stream())


def im2row(image, patches, P, gh, gw) -> None:
    B, C, H, W = image.shape
    _chk(image, F32, 'im2row image')
    hip.call('crl_im2row', _p(image), _p(patches), B, C, H, W, P, gh, gw, patches.shape[1], _stream())


def vit_tokens_fwd(patch, cls, pos, x, B, Np, D) -> None:
    hip.call('crl_vit_tokens_fwd', _p(patch), _p(cls), _p(pos), _p(x), B, Np, D, _stream())


def vit_tokens_bwd(dx, dpatch, dcls, dpos, B, Np, D, accumulate: bool = True) -> None:
    hip.call('crl_vit_tokens_bwd', _p(dx), _p(dpatch), _p(dcls), _p(dpos), int(accumulate), B, Np, D, _stream())


def embed_fwd(ids, tok, pos, out, pos_offset: int = 2) -> None:
    B, T = ids.shape
    hip.call('crl_embed_fwd', _p(ids), _p(tok), _p(pos), _p(out), B, T, out.shape[1], pos_offset, tok.shape[0], _stream())


def embed_bwd(ids, dt, dtok, dpos, pos_offset: int = 2, accumulate: bool = True) -> None:
    B, T = ids.shape
    nbytes = hip.query('crl_embed_bwd_ws_bytes', B, T, dt.shape[1])
    ws = _scratch.get(nbytes, dt.device)
    hip.call('crl_embed_bwd', _p(ids), _p(dt), _p(dtok), _p(dpos), int(accumulate), B, T, dt.shape[1], pos_offset, dtok.shape[0],
             _p(ws), nbytes, _stream())


def cross_entropy(logits, target, V: int, loss_mul: float, grad_mul: float, loss, n_valid, row_loss, dlogits,
                  grad_mul_dev: Optional[torch.Tensor] = None) -> None:
    """grad_mul_dev: device fp32 scalar multiplied into the gradient on the device (the GradScaler loss scale)"""
    M = logits.shape[0]
    hip.call('crl_cross_entropy', _p(logits), logits.stride(0), _p(target), M, V, float(loss_mul), float(grad_mul), _p(grad_mul_dev),
             _p(loss), _p(n_valid), _p(row_loss), _p(dlogits), _stream())


def _rows_ok(M: int, index: int, *rows) -> bool:
    return all(t is None or (t.dtype is F32 and t.shape == (M,) and t.is_contiguous() and t.get_device() == index) for t in rows)


def _logits_ok(logits, target, V: int, M: int, ld: int, index: int) -> bool:
    f32 = logits.dtype is F32
    vec = 4 if f32 else 8
    return (index >= 0 and (f32 or logits.dtype is BF16) and logits.dim() == 2 and 0 < V <= logits.shape[1] and logits.stride(1) == 1
            and (M == 1 or (ld % vec == 0 and ld >= logits.shape[1]))
            and (target is None or (target.dtype is torch.int64 and target.shape == (M,) and target.is_contiguous() and target.get_device() == index)))


def _want_aligned_rows(t: torch.Tensor, name: str) -> None:
    ld = t.stride(0)
    if t.shape[0] > 1 and (ld % (16 // t.element_size()) or ld < t.shape[1]):
        raise ValueError(f'{name}: rows {ld} elements apart; every row must start at a 16-byte boundary behind the one before (pad the rows)')


def _refuse_logits(logits, target, V: int, **rows) -> None:
    if logits.dtype not in (BF16, F32):
        raise TypeError(f'logits: expected bf16 or fp32, got {logits.dtype}')
    _want(logits, 'logits', logits.dtype, None, None)
    if not 0 < V <= logits.shape[1]:
        raise ValueError(f'logits: {logits.shape[1]} columns, V = {V}')
    M = logits.shape[0]
    _want_aligned_rows(logits, 'logits')
    _want(target, 'target', torch.int64, M)
    if target is not None and not target.is_contiguous():
        raise ValueError('target must be contiguous')
    for name, t in rows.items():
        _want(t, name, F32, M)
        if t is not None and not t.is_contiguous():
            raise ValueError(f'{name} must be contiguous')


def token_logprobs(logits, target, V: int, logprob, entropy: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   top_logprob: Optional[torch.Tensor] = None, top_ids: Optional[torch.Tensor] = None) -> None:
    """per row of logits [M, >= V] (bf16 or fp32, rows that start at 16-byte boundaries; the first V columns count): logprob [M] fp32 = log softmax at target
    [M] int64 (-100: 0; outside the vocabulary: NaN), entropy [M] (nats), lse [M] = log sum exp, and the k <= 32 most probable tokens, falling, of
    equal ones the lower first: top_ids [M, k] int64, top_logprob [M, k] fp32.  Whatever is None is left out (logprob and target together)."""
    M, ld, index = logits.shape[0], logits.stride(0), logits.get_device()
    k, ls, is_ = (top_ids.shape[-1], top_logprob.stride(), top_ids.stride()) if top_ids is not None and top_logprob is not None else (0, (0, 1), (0, 1))
    if not (_logits_ok(logits, target, V, M, ld, index) and _rows_ok(M, index, logprob, entropy, lse) and (target is None) == (logprob is None)
            and (top_ids is None) == (top_logprob is None)
            and (top_ids is None or (top_ids.shape == (M, k) == top_logprob.shape and 1 <= k <= min(32, V) and top_ids.dtype is torch.int64
                                     and top_logprob.dtype is F32 and ls[1] == 1 == is_[1] and min(ls[0], is_[0]) >= k
                                     and top_ids.get_device() == index == top_logprob.get_device()))
            and not (logprob is None and entropy is None and lse is None and top_ids is None)):
        _refuse_logprobs(logits, target, V, logprob, entropy, lse, top_logprob, top_ids)
    _run_on(index, 'crl_token_logprobs', logits.data_ptr(), int(logits.dtype is F32), ld, _p(target), M, V, _p(logprob), _p(entropy), _p(lse), k,
            _p(top_logprob), ls[0], _p(top_ids), is_[0])


def _refuse_logprobs(logits, target, V, logprob, entropy, lse, top_logprob, top_ids):
    def shapes():
        _refuse_logits(logits, target, V, logprob=logprob, entropy=entropy, lse=lse)
        if (target is None) != (logprob is None):
            raise ValueError('logprob and target go together')
        if (top_ids is None) != (top_logprob is None):
            raise ValueError('top_ids and top_logprob go together')
        if logprob is None and entropy is None and lse is None and top_ids is None:
            raise ValueError('nothing to compute')
        if top_ids is not None:
            _want(top_ids, 'top_ids', torch.int64, logits.shape[0], None)
            k = top_ids.shape[1]
            _want(top_logprob, 'top_logprob', F32, logits.shape[0], k)
            if not 1 <= k <= min(32, V):
                raise ValueError(f'top_ids: {k} of {V} tokens; 1 to 32 are possible')
            _want_rows(top_ids, 'top_ids', k)
            _want_rows(top_logprob, 'top_logprob', k)
    _refuse(('logits', 'target', 'logprob', 'entropy', 'lse', 'top_logprob', 'top_ids'), locals(), shapes)


def token_logprobs_bwd(logits, target, V: int, lse, entropy, d_logprob, d_entropy, dlogits) -> None:
    """gradient of token_logprobs: dlogits (like logits; may be logits itself) = d_logprob (onehot(target) - p) - d_entropy p (log p + entropy) per
    row, its columns from V on zeroed.  lse, entropy [M]: what the forward call gave; d_logprob, d_entropy
    [M]: one of them may be None.  A target of -100 takes no d_logprob; rows that take neither gradient become zeros, whatever their logits are."""
    M, ld, ldd, index = logits.shape[0], logits.stride(0), dlogits.stride(0), logits.get_device()
    cols = dlogits.shape[-1]
    if not (_logits_ok(logits, target, V, M, ld, index) and _logits_ok(dlogits, None, V, M, ldd, index) and dlogits.shape == logits.shape
            and dlogits.dtype is logits.dtype
            and _rows_ok(M, index, lse, entropy, d_logprob, d_entropy) and lse is not None and not (d_logprob is None and d_entropy is None)
            and (d_logprob is None or target is not None) and (d_entropy is None or entropy is not None)):
        _refuse_logprobs_bwd(logits, target, V, lse, entropy, d_logprob, d_entropy, dlogits)
    _run_on(index, 'crl_token_logprobs_bwd', logits.data_ptr(), int(logits.dtype is F32), ld, _p(target), M, V, lse.data_ptr(), _p(entropy),
            _p(d_logprob), _p(d_entropy), dlogits.data_ptr(), ldd, cols)


def _refuse_logprobs_bwd(logits, target, V, lse, entropy, d_logprob, d_entropy, dlogits):
    def shapes():
        if d_logprob is None and d_entropy is None:
            raise ValueError('neither d_logprob nor d_entropy')
        if (d_logprob is not None and target is None) or (d_entropy is not None and entropy is None) or lse is None:
            raise ValueError('d_logprob needs target, d_entropy needs entropy, and lse is needed')
        _refuse_logits(logits, target, V, lse=lse, entropy=entropy, d_logprob=d_logprob, d_entropy=d_entropy)
        _want(dlogits, 'dlogits', logits.dtype, *logits.shape)
        _want_aligned_rows(dlogits, 'dlogits')
    _refuse(('logits', 'target', 'lse', 'entropy', 'd_logprob', 'd_entropy', 'dlogits'), locals(), shapes)


def grad_norm(g, max_norm: float, inv_scale: float, state) -> None:
    ws = _scratch.get(hip.query('crl_grad_norm_ws_bytes'), g.device)
    hip.call('crl_grad_norm', _p(g), g.numel(), float(max_norm), float(inv_scale), _p(state), _p(ws), _stream())


def grad_norm_scaled(g, max_norm: float, grad_divisor: float, growth_factor: float, backoff_factor: float, growth_interval: int,
                     state) -> None:
    """unscale + inf check + clip coefficient + GradScaler.update() on the device (state: 8 floats, scale in state[4])"""
    assert state.numel() >= 8
    ws = _scratch.get(hip.query('crl_grad_norm_ws_bytes'), g.device)
    hip.call('crl_grad_norm_scaled', _p(g), g.numel(), float(max_norm), float(grad_divisor), float(growth_factor), float(backoff_factor),
             int(growth_interval), _p(state), _p(ws), _stream())


def optim_prepare(state, base_lr: float, warmup_lr_init: float, lr_min: float, warmup_t: int, t_initial: int, beta1: float, beta2: float) -> None:
    """device-side learning rate (state[8], cosine + warm-up at state[7] updates; t_initial <= 0: constant) and bias corrections (state[9], [10])"""
    assert state.numel() >= 16
    hip.call('crl_optim_prepare', _p(state), float(base_lr), float(warmup_lr_init), float(lr_min), int(warmup_t), int(t_initial),
             float(beta1), float(beta2), _stream())


def adamw(p, g, m, v, p_bf16, lr, beta1, beta2, eps, weight_decay, step: int, state, zero_grad: bool) -> None:
    """step >= 1: host-side step number; step == 0: device-side mode (bias corrections, and the learning rate when lr < 0, from the
    state words written by optim_prepare)"""
    hip.call('crl_adamw', _p(p), _p(g), _p(m), _p(v), _p(p_bf16), p.numel(), float(lr), float(beta1), float(beta2),
             float(eps), float(weight_decay), int(step), _p(state), int(zero_grad), _stream())


def cast_bf16(src, dst) -> None:
    hip.call('crl_cast_bf16', _p(src), _p(dst), src.numel(), _stream())


def cast_pad_bf16(src, dst, R: int, C: int, Cp: int) -> None:
    hip.call('crl_cast_pad_bf16', _p(src), _p(dst), R, C, Cp, _stream())


class DropSpec:
    """(p, seed, step) of one forward / backward pair; site ids are chosen by the caller (one per dropout call site)"""

    def __init__(self, p: float, seed: int, step: int, p_attn: float = 0.0, p_act: float = 0.0, p_path: float = 0.0):
        """p: hidden-state dropout; p_attn: attention-probability dropout; p_act: activation (post-GELU) dropout; p_path: the
        encoder's maximum drop-path rate (Swin: per block linearly from 0 to p_path)"""
        self.p, self.seed, self.step = float(p), int(seed) & (2 ** 64 - 1), int(step) & (2 ** 32 - 1)
        self.p_attn, self.p_act, self.p_path = float(p_attn), float(p_act), float(p_path)


def dropout(x: torch.Tensor, y: torch.Tensor, d: DropSpec, site: int, y_bf16: Optional[torch.Tensor] = None, p: Optional[float] = None) -> None:
    """y = dropout(x) (bf16 or fp32, in place allowed); fp32 inputs may emit a bf16 copy of the result. p overrides d.p (activation dropout)"""
    assert x.dtype == y.dtype and x.is_contiguous() and y.is_contiguous()
    hip.call('crl_dropout', _p(x), _p(y), x.numel(), int(x.dtype == F32), _p(y_bf16), d.p if p is None else float(p), d.seed, d.step, site, _stream())


def droppath_scale(scale: torch.Tensor, p: float, d: DropSpec, site: int) -> None:
    """scale[b] = keep(b) / (1 - p): one drop-path decision per sample for (d.seed, d.step, site)"""
    _chk(scale, F32, 'droppath scale')
    hip.call('crl_droppath_scale', _p(scale), scale.numel(), float(p), d.seed, d.step, site, _stream())


def rowscale_add(x_bf16: torch.Tensor, scale: torch.Tensor, resid: torch.Tensor, out: torch.Tensor, rows_per_sample: int) -> None:
    """out(f32) = resid + bf16(x * scale[sample of the row])"""
    M, C = x_bf16.shape
    assert x_bf16.is_contiguous() and resid.is_contiguous() and out.is_contiguous()
    hip.call('crl_rowscale_add', _p(x_bf16), _p(scale), _p(resid), _p(out), M, int(rows_per_sample), C, _stream())


def rowscale_bf16(x_bf16: torch.Tensor, scale: torch.Tensor, y_bf16: torch.Tensor, rows_per_sample: int) -> None:
    M, C = x_bf16.shape
    assert x_bf16.is_contiguous() and y_bf16.is_contiguous()
    hip.call('crl_rowscale_bf16', _p(x_bf16), _p(scale), _p(y_bf16), M, int(rows_per_sample), C, _stream())


def dropout_add(x_bf16: torch.Tensor, resid: torch.Tensor, out: torch.Tensor, d: DropSpec, site: int) -> None:
    """out(f32) = resid(f32) + bf16(dropout(x_bf16))"""
    _chk(x_bf16, BF16, 'dropout_add x')
    _chk(resid, F32, 'dropout_add resid')
    assert x_bf16.is_contiguous() and resid.is_contiguous() and out.is_contiguous()
    hip.call('crl_dropout_add', _p(x_bf16), _p(resid), _p(out), x_bf16.numel(), d.p, d.seed, d.step, site, _stream())


def dropout_mask(n: int, d: DropSpec, site: int, device, p: Optional[float] = None) -> torch.Tensor:
    keep = torch.empty(n, dtype=torch.uint8, device=device)
    hip.call('crl_dropout_mask', _p(keep), n, d.p if p is None else float(p), d.seed, d.step, site, _stream())
    return keep


def add_bf16_to_f32(x_bf16, y, accumulate: bool) -> None:
    hip.call('crl_add_bf16_to_f32', _p(x_bf16), _p(y), x_bf16.numel(), int(accumulate), _stream())


# ------------------------------------------------------------------------------------------- measurement aids
def gemm_set_schedule(dynamic: bool) -> None:
    """persistent GEMMs: dynamic tile tickets (default) or the static tile walk (A/B runs, tests); results are bit-identical"""
    hip.call('crl_gemm_set_schedule', int(bool(dynamic)))


def gemm_set_reserved_cus(n: int) -> None:
    """persistent GEMMs launch on 256 - n CUs (the rest is left to RCCL's kernels while gradient buckets are in flight)"""
    hip.call('crl_gemm_set_reserved_cus', int(n))


class OccupyCUs:
    """`with OccupyCUs(n):` -- n CUs are held by a sleeping side-stream kernel (crl_debug_occupy_cus) for the duration of the block:
    the single-GPU stand-in for the CUs RCCL's all-reduce kernels take from the training step of a data-parallel run.
    Inside the block wait for work with `torch.cuda.current_stream().synchronize()`: a device-wide synchronize waits for the sleepers."""

    def __init__(self, n_cus: int, max_seconds: float = 60.0):
        self.n, self.max_seconds = int(n_cus), float(max_seconds)

    def __enter__(self):
        import time
        self.flag = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        hip.call('crl_debug_occupy_cus', self.n, self.max_seconds, self.flag.data_ptr(), self.stream.cuda_stream)
        time.sleep(0.02)          # the sleepers are resident before the disturbed work is enqueued
        return self

    def __exit__(self, *exc):
        self.flag[0] = 1
        self.stream.synchronize()
        return False
