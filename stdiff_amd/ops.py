"""Tensor-level wrappers over the C ABI (one function per entry point of include/stdiff_hip.h).
Tensors must live on the GPU; outputs are allocated with torch when not supplied."""
import ctypes as C
import operator

import numpy as np
import torch

from . import _lib as L
from ._lib import F32, check, dt_of, lib, lib_for, ptr, require_gpu, stream


def round_up(a, b):
    return (a + b - 1) // b * b


def gemm(A, W, bias=None, out=None, out_dtype=None, epi=L.EPI_BIAS, gate=None, res=None, out2=None, M=None,
         workspace=None, a_kmajor=False, w_kmajor=False, static_scratch=False, ln_parts=None, stats_out=None,
         defer=None):
    """out[M,N] = epi(A[M,K] @ W[N,K]^T + bias). A/W: same dtype (fp32 or bf16), K-contiguous rows -- or, with
    a_kmajor / w_kmajor, given as [K, M] / [K, N] (K rows; need not be a multiple of the K-slab).
    static_scratch=True: stdiff_gemm_static_scratch -- split-K partials in the library's own device array, nothing is
    allocated by the library (`out` must be given for the CALLER not to allocate either).
    defer: an L.SplitResult; when the launch splits K (bias / gated-residual epilogues only) the reduce launch is skipped
    and `defer` describes the partial products for a *_split consumer (defer.slices == 0: `out` is complete)."""
    require_gpu(A, W, bias, out, gate, res, out2, workspace)
    bk = 64 if A.element_size() == 2 else 16
    kA = A.shape[0] if a_kmajor else A.shape[1]
    kW = W.shape[0] if w_kmajor else W.shape[1]
    if a_kmajor and w_kmajor:
        assert kA == kW
        k_valid, K = kA, round_up(kA, bk)
    elif a_kmajor or w_kmajor:
        k_valid = kA if a_kmajor else kW            # the row-major operand carries the (zero-)padded K
        K = kW if a_kmajor else kA
        assert k_valid <= K, (k_valid, K)
    else:
        assert kA == kW
        k_valid = K = kA
    M = (A.shape[1] if a_kmajor else A.shape[0]) if M is None else M
    N = W.shape[1] if w_kmajor else W.shape[0]
    if out is None:
        out = torch.empty((M, N // 2 if epi == L.EPI_LN_MOD else N), device=A.device, dtype=out_dtype or A.dtype)
    a = L.GemmArgs()
    a.M, a.N, a.K = M, N, K
    a.a_layout, a.w_layout, a.k_valid = int(a_kmajor), int(w_kmajor), k_valid
    a.A, a.lda, a.a_dtype = ptr(A), A.stride(0), dt_of(A)
    a.W, a.ldw = ptr(W), W.stride(0)
    a.bias = ptr(bias)
    a.C, a.ldc, a.c_dtype = ptr(out), out.stride(0), dt_of(out)
    a.epi = epi
    if gate is not None:
        a.gate, a.ldgate = ptr(gate), gate.stride(0)
    if res is not None:
        a.res, a.ldres = ptr(res), res.stride(0)
    if out2 is not None:
        a.C2, a.ldc2 = ptr(out2), out2.stride(0)
    if ln_parts is not None:           # EPI_LN_MOD: partial row moments of `res`, fp32 [M, parts, 2] (row_stats: 1 part)
        require_gpu(ln_parts)
        assert ln_parts.dtype == torch.float32 and ln_parts.is_contiguous() and ln_parts.shape[0] >= M
        a.ln_parts, a.ln_nparts = ptr(ln_parts), ln_parts.shape[1]
    if stats_out is not None:          # gated-residual epilogue also writes the partial row moments of its output
        require_gpu(stats_out)
        assert stats_out.dtype == torch.float32 and stats_out.is_contiguous() and stats_out.shape == (M, N // 256, 2)
        a.stats_out = ptr(stats_out)
    if workspace is not None:          # fp32 scratch for split-K (small outputs with a long K)
        a.workspace, a.workspace_bytes = ptr(workspace), workspace.numel() * workspace.element_size()
    if defer is not None:
        a.defer = C.pointer(defer)
    lb = lib_for(A, W, out, gate, out2)
    check((lb.stdiff_gemm_static_scratch if static_scratch else lb.stdiff_gemm)(C.byref(a), stream()))
    return out


def _dw_group_args(problems, C_rows):
    a = L.DwGroupArgs()
    assert 1 <= len(problems) <= 8
    first = problems[0][0]
    a.n, a.C, a.dtype = len(problems), first.shape[0] if C_rows is None else C_rows, dt_of(first)
    for i, pr in enumerate(problems):
        dY, X, gw, gb = pr[:4]
        require_gpu(dY, X, gw, gb)
        assert dY.dtype == first.dtype and X.dtype == first.dtype and gw.dtype == torch.float32 and gw.is_contiguous()
        assert dY.shape[0] >= a.C and X.shape[0] >= a.C and dY.stride(1) == 1 and X.stride(1) == 1
        q = a.p[i]
        q.M, q.N = (gw.shape[0] if len(pr) < 5 or pr[4] is None else pr[4]), gw.shape[1]
        assert dY.shape[1] >= q.M and X.shape[1] >= q.N
        q.dY, q.lddy, q.X, q.ldx = ptr(dY), dY.stride(0), ptr(X), X.stride(0)
        q.gw, q.ldgw, q.gb = ptr(gw), gw.stride(0), ptr(gb)
    return a, first


def dw_group_parts(problems, C_rows=None):
    """Number of floats dw_group(problems, sq_parts=...) writes."""
    a, first = _dw_group_args(problems, C_rows)
    n = lib_for(first).stdiff_dw_group_parts(C.byref(a))
    if n < 0:
        raise ValueError("stdiff_dw_group_parts: bad problem list")
    return int(n)


def dw_group(problems, C_rows=None, sq_parts=None):
    """One launch for several weight gradients over the same batch: for each (dY, X, gw, gb[, M]) in `problems`
    gw[M, N] = dY[:, :M]^T X[:, :N] and gb[M] = colsum(dY[:, :M]) (gb may be None).  dY [C, >= M], X [C, >= N] of the
    operand dtype, gw / gb fp32, overwritten.  sq_parts (fp32 [>= dw_group_parts(problems)], optional): overwritten with
    per-wave sums of squares of everything written -- their sum is the launch's squared gradient norm (sum_parts)."""
    a, first = _dw_group_args(problems, C_rows)
    if sq_parts is not None:
        require_gpu(sq_parts)
        n = lib_for(first).stdiff_dw_group_parts(C.byref(a))
        assert sq_parts.dtype == torch.float32 and sq_parts.is_contiguous() and 0 <= n <= sq_parts.numel()
        a.sq_parts = ptr(sq_parts)
    check(lib_for(first).stdiff_dw_group(C.byref(a), stream()))


def sum_parts(parts, out, accumulate=True):
    """out[0] (+)= parts.sum(), one workgroup, fixed order (the same bits every run)."""
    require_gpu(parts, out)
    assert parts.dtype == torch.float32 and out.dtype == torch.float32 and parts.is_contiguous()
    check(lib().stdiff_sum_parts(ptr(parts), parts.numel(), ptr(out), int(accumulate), stream()))


def transpose(x, out=None, rows_pad=None):
    """out[c, r] = x[r, c]; columns rows..rows_pad-1 of out are zero-filled (K padding of the backward GEMMs)."""
    require_gpu(x, out)
    r, c = x.shape
    rows_pad = r if rows_pad is None else rows_pad
    if out is None:
        out = torch.empty((c, rows_pad), device=x.device, dtype=x.dtype)
    check(lib_for(x, out).stdiff_transpose(ptr(x), x.stride(0), ptr(out), out.stride(0), r, c, rows_pad, dt_of(x), stream()))
    return out


def attention_fwd(qkv, cu_rows, max_chunk, heads, out=None, lse=None):
    """qkv [R,3H] -> out [R,H]; cu_rows int32 device [n_chunks+1]."""
    require_gpu(qkv, cu_rows, out, lse)
    R, H3 = qkv.shape
    H = H3 // 3
    if out is None:
        out = torch.empty((R, H), device=qkv.device, dtype=qkv.dtype)
    check(lib_for(qkv, out).stdiff_attention_fwd(ptr(qkv), qkv.stride(0), ptr(out), out.stride(0), ptr(lse), ptr(cu_rows),
                                     cu_rows.numel() - 1, max_chunk, heads, H // heads, dt_of(qkv), stream()))
    return out


def ln_modulate(x, shift, scale, out=None, out_dtype=None, mean=None, rstd=None, split=None, bias=None, gate=None,
                res=None, v_out=None):
    """LayerNorm(x, eps=1e-6, no affine) * (1 + scale) + shift; shift/scale are column views of the adaLN output.
    split (an L.SplitResult with slices > 1): x is not read but FORMED first -- v = sum of the slices + bias,
    x = res + gate * v (x = v without a gate), v_out = v -- and written (stdiff_ln_modulate_split)."""
    require_gpu(x, shift, scale, out, bias, gate, res, v_out)
    R, H = x.shape
    assert shift.stride(0) == scale.stride(0) and shift.dtype == scale.dtype
    if out is None:
        out = torch.empty((R, H), device=x.device, dtype=out_dtype or shift.dtype)
    if split is not None and split.slices > 1:
        check(lib_for(shift, out).stdiff_ln_modulate_split(
            C.byref(split), ptr(bias), ptr(gate), gate.stride(0) if gate is not None else 0, ptr(res),
            res.stride(0) if res is not None else 0, ptr(x), x.stride(0), ptr(v_out),
            v_out.stride(0) if v_out is not None else 0, ptr(shift), ptr(scale), shift.stride(0), dt_of(shift), ptr(out),
            out.stride(0), dt_of(out), ptr(mean), ptr(rstd), R, H, stream()))
        return out
    check(lib_for(shift, out).stdiff_ln_modulate(ptr(x), x.stride(0), ptr(shift), ptr(scale), shift.stride(0), dt_of(shift),
                                   ptr(out), out.stride(0), dt_of(out), ptr(mean), ptr(rstd), R, H, stream()))
    return out


def row_stats(x, parts=None):
    """Row moments of x fp32 [R, H] as ONE part per row: fp32 [R, 1, 2] = (mean, sum of squared deviations) -- the
    statistics of LayerNorm(eps 1e-6, biased variance) in the form the LN_MOD GEMM epilogue reads."""
    require_gpu(x, parts)
    R, H = x.shape
    if parts is None:
        parts = torch.empty((R, 1, 2), device=x.device, dtype=torch.float32)
    assert parts.dtype == torch.float32 and parts.is_contiguous() and parts.numel() >= 2 * R
    check(lib().stdiff_row_stats(ptr(x), x.stride(0), ptr(parts), R, H, stream()))
    return parts


def silu_cond(ycond, temb=None, t_index=None, out=None, out_dtype=torch.float32):
    require_gpu(ycond, temb, t_index, out)
    R, H = ycond.shape
    if out is None:
        out = torch.empty((R, H), device=ycond.device, dtype=out_dtype)
    check(lib_for(out).stdiff_silu_cond(ptr(temb), ptr(t_index), ptr(ycond), ycond.stride(0), ptr(out), out.stride(0),
                                 dt_of(out), R, H, stream()))
    return out


def timestep_embedding(t, freqs, out=None, out_dtype=torch.float32):
    require_gpu(t, freqs, out)
    assert t.dtype == torch.int64
    R = t.numel()
    if out is None:
        out = torch.empty((R, 256), device=t.device, dtype=out_dtype)
    check(lib_for(out).stdiff_timestep_embedding(ptr(t), ptr(freqs), ptr(out), out.stride(0), dt_of(out), R, stream()))
    return out


def pack_rows(src, cpad, dtype, out=None):
    require_gpu(src, out)
    R, Cc = src.shape
    if out is None:
        out = torch.empty((R, cpad), device=src.device, dtype=dtype)
    check(lib_for(out).stdiff_pack_rows(ptr(src), src.stride(0), ptr(out), out.stride(0), dt_of(out), R, Cc, cpad, stream()))
    return out


def gather_rows2(a, b, idx, out_a=None, out_b=None):
    """(a[idx], b[idx]) for fp32 [N, C] matrices on the device and an int64 device index vector (b may be None)."""
    require_gpu(a, b, idx, out_a, out_b)
    R, Cc = idx.shape[0], a.shape[1]
    assert idx.dtype == torch.int64 and a.dtype == torch.float32 and (b is None or (b.dtype == a.dtype and b.shape == a.shape))
    if out_a is None:
        out_a = torch.empty((R, Cc), device=a.device, dtype=torch.float32)
    if b is not None and out_b is None:
        out_b = torch.empty((R, Cc), device=a.device, dtype=torch.float32)
    check(lib().stdiff_gather_rows2(ptr(a), a.stride(0), ptr(b), b.stride(0) if b is not None else 0, ptr(idx),
                                    ptr(out_a), out_a.stride(0), ptr(out_b), out_b.stride(0) if b is not None else 0,
                                    R, Cc, stream()))
    return out_a, out_b


def ddpm_step(x, eps, gt, mask, coef, t_dev, t_first, z_base=None, seed=0, row_offset=0, xp=None, pred_type=0, z_rows=0):
    require_gpu(x, eps, gt, mask, coef, t_dev, z_base, xp)
    a = L.StepArgs()
    a.x, a.eps, a.gt, a.mask, a.coef = ptr(x), ptr(eps), ptr(gt), ptr(mask), ptr(coef)
    a.t_dev, a.t_first = ptr(t_dev), t_first
    a.z_base, a.seed, a.row_offset = ptr(z_base), seed, row_offset
    if xp is not None:
        a.xp, a.ldxp, a.xp_dtype = ptr(xp), xp.stride(0), dt_of(xp)
    a.R, a.G, a.pred_type, a.z_rows = x.shape[0], x.shape[1], pred_type, int(z_rows)
    check(lib_for(xp).stdiff_ddpm_step(C.byref(a), stream()))


def advance_timestep(t_dev):
    check(lib().stdiff_advance_timestep(ptr(t_dev), stream()))


def spin_probe(blocks, microseconds):
    """`blocks` idle one-wave workgroups for `microseconds` on the current stream (stream-concurrency probe)."""
    check(lib().stdiff_spin_probe(int(blocks), int(microseconds), stream()))


def init_sample(x, gt, mask, z=None, seed=0, row_offset=0, xp=None):
    require_gpu(x, gt, mask, z, xp)
    check(lib_for(xp).stdiff_init_sample(ptr(x), ptr(z), seed, row_offset, ptr(gt), ptr(mask), ptr(xp),
                                   xp.stride(0) if xp is not None else 0, dt_of(xp) if xp is not None else F32,
                                   x.shape[0], x.shape[1], stream()))


def add_noise_splice(x, noise, t, sqrt_ac, sqrt_1mac, mask, x_noisy=None, xp=None):
    require_gpu(x, noise, t, sqrt_ac, sqrt_1mac, mask, x_noisy, xp)
    check(lib_for(xp).stdiff_add_noise_splice(ptr(x), ptr(noise), ptr(t), ptr(sqrt_ac), ptr(sqrt_1mac), ptr(mask),
                                        ptr(x_noisy), ptr(xp), xp.stride(0) if xp is not None else 0,
                                        dt_of(xp) if xp is not None else F32, x.shape[0], x.shape[1], stream()))


def masked_mse(pred, noise, mask, loss, dpred=None, dp=None, grad_scale=1.0):
    require_gpu(pred, noise, mask, loss, dpred, dp)
    check(lib_for(dp).stdiff_masked_mse(ptr(pred), ptr(noise), ptr(mask), ptr(loss), ptr(dpred), ptr(dp),
                                  dp.stride(0) if dp is not None else 0, dt_of(dp) if dp is not None else F32,
                                  grad_scale, pred.shape[0], pred.shape[1], stream()))


def attention_bwd(qkv, out, dout, lse, cu_rows, max_chunk, heads, dqkv=None, delta=None, split=None):
    """split (an L.SplitResult with slices > 1): dout is first FORMED from the partial products (and written)."""
    require_gpu(qkv, out, dout, lse, cu_rows, dqkv, delta)
    R, H3 = qkv.shape
    H = H3 // 3
    if dqkv is None:
        dqkv = torch.empty_like(qkv)
    if delta is None:
        delta = torch.empty((R, heads), device=qkv.device, dtype=torch.float32)
    if split is not None and split.slices > 1:
        check(lib_for(qkv, out, dout, dqkv).stdiff_attention_bwd_split(
            ptr(qkv), qkv.stride(0), ptr(out), out.stride(0), C.byref(split), ptr(dout), dout.stride(0), ptr(lse),
            ptr(delta), ptr(dqkv), dqkv.stride(0), ptr(cu_rows), cu_rows.numel() - 1, max_chunk, R, heads, H // heads,
            dt_of(qkv), stream()))
        return dqkv
    check(lib_for(qkv, out, dout, dqkv).stdiff_attention_bwd(ptr(qkv), qkv.stride(0), ptr(out), out.stride(0), ptr(dout), dout.stride(0),
                                     ptr(lse), ptr(delta), ptr(dqkv), dqkv.stride(0), ptr(cu_rows),
                                     cu_rows.numel() - 1, max_chunk, R, heads, H // heads, dt_of(qkv), stream()))
    return dqkv


def ln_modulate_bwd(dy, x, mean, rstd, scale, dx, dshift, dscale, accumulate=True, gate=None, branch=None, dbranch=None,
                    dgate=None, split=None):
    """LayerNorm + modulate backward; with gate / branch / dbranch / dgate also the gated-residual backward of the
    branch below it on the finished dx row (dbranch = dx * gate, dgate = dx * branch): one launch instead of two."""
    require_gpu(dy, x, mean, rstd, scale, dx, dshift, dscale, gate, branch, dbranch, dgate)
    R, H = x.shape
    assert dshift.stride(0) == dscale.stride(0)
    lb = lib_for(dy, scale, dshift)
    if split is not None and split.slices > 1:       # dy = the partial products summed (and rounded to the dtype)
        z = lambda t_: t_.stride(0) if t_ is not None else 0
        check(lb.stdiff_ln_modulate_bwd_split(C.byref(split), dt_of(scale), ptr(x), x.stride(0), ptr(mean), ptr(rstd),
                                              ptr(scale), scale.stride(0), ptr(dx), dx.stride(0), int(accumulate),
                                              ptr(dshift), ptr(dscale), dshift.stride(0), ptr(gate), z(gate), ptr(branch),
                                              z(branch), ptr(dbranch), z(dbranch), ptr(dgate), z(dgate), R, H, stream()))
        return
    if gate is None:
        check(lb.stdiff_ln_modulate_bwd(ptr(dy), dy.stride(0), dt_of(dy), ptr(x), x.stride(0), ptr(mean), ptr(rstd),
                                        ptr(scale), scale.stride(0), ptr(dx), dx.stride(0), int(accumulate),
                                        ptr(dshift), ptr(dscale), dshift.stride(0), R, H, stream()))
        return
    check(lb.stdiff_ln_modulate_bwd_gate(ptr(dy), dy.stride(0), dt_of(dy), ptr(x), x.stride(0), ptr(mean), ptr(rstd),
                                         ptr(scale), scale.stride(0), ptr(dx), dx.stride(0), int(accumulate),
                                         ptr(dshift), ptr(dscale), dshift.stride(0), ptr(gate), gate.stride(0),
                                         ptr(branch), branch.stride(0), ptr(dbranch), dbranch.stride(0), ptr(dgate),
                                         dgate.stride(0), R, H, stream()))


def gate_bwd(dh, gate, branch, dbranch, dgate):
    require_gpu(dh, gate, branch, dbranch, dgate)
    R, H = dh.shape
    check(lib_for(gate, branch, dbranch, dgate).stdiff_gate_bwd(ptr(dh), dh.stride(0), ptr(gate), gate.stride(0), ptr(branch), branch.stride(0),
                                ptr(dbranch), dbranch.stride(0), ptr(dgate), dgate.stride(0), dt_of(gate), R, H,
                                stream()))


def gelu_bwd(dg, u_pre, du):
    require_gpu(dg, u_pre, du)
    R, Cc = dg.shape
    assert dg.stride(0) == u_pre.stride(0) == du.stride(0)
    check(lib_for(dg, u_pre, du).stdiff_gelu_bwd(ptr(dg), ptr(u_pre), ptr(du), dg.stride(0), dt_of(dg), R, Cc, stream()))


def silu_bwd(ds, c, dc, accumulate=False):
    require_gpu(ds, c, dc)
    R, H = ds.shape
    check(lib_for(ds, c, dc).stdiff_silu_bwd(ptr(ds), ds.stride(0), dt_of(ds), ptr(c), c.stride(0), dt_of(c), ptr(dc),
                                dc.stride(0), dt_of(dc), int(accumulate), R, H, stream()))


def colsum(dY, db, accumulate=False):
    require_gpu(dY, db)
    R, Cc = dY.shape
    check(lib_for(dY).stdiff_colsum(ptr(dY), dY.stride(0), dt_of(dY), ptr(db), int(accumulate), R, Cc, stream()))


def grad_sumsq(g, sumsq):
    require_gpu(g, sumsq)
    check(lib().stdiff_grad_sumsq(ptr(g), g.numel(), ptr(sumsq), stream()))


def adamw_args(p, g, m, v, sumsq, step_dev, scal, lr, max_norm=1.0, grad_scale=1.0, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.0, bf16_mirror=None):
    """stdiff_adamw_args over the flat buffers (for adamw_prepare / adamw_range: the update issued range by range)."""
    require_gpu(p, g, m, v, sumsq, step_dev, scal, bf16_mirror)
    a = L.AdamWArgs()
    a.params, a.grads, a.exp_avg, a.exp_avg_sq, a.n = ptr(p), ptr(g), ptr(m), ptr(v), p.numel()
    a.sumsq, a.step_dev, a.scal = ptr(sumsq), ptr(step_dev), ptr(scal)
    a.max_norm, a.grad_scale, a.lr = max_norm, grad_scale, lr
    a.beta1, a.beta2, a.eps, a.weight_decay = betas[0], betas[1], eps, weight_decay
    if bf16_mirror is not None:
        assert bf16_mirror.dtype == torch.bfloat16 and bf16_mirror.numel() == p.numel()
        a.bf16_mirror = ptr(bf16_mirror)
    return a


def adamw_prepare(a):
    check(lib().stdiff_adamw_prepare(C.byref(a), stream()))


def adamw_range(a, lo, count):
    check(lib().stdiff_adamw_range(C.byref(a), lo, count, stream()))


def clip_adamw(p, g, m, v, sumsq, step_dev, scal, lr, max_norm=1.0, grad_scale=1.0, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.0, bf16_mirror=None):
    require_gpu(p, g, m, v, sumsq, step_dev, scal, bf16_mirror)
    a = L.AdamWArgs()
    a.params, a.grads, a.exp_avg, a.exp_avg_sq, a.n = ptr(p), ptr(g), ptr(m), ptr(v), p.numel()
    a.sumsq, a.step_dev, a.scal = ptr(sumsq), ptr(step_dev), ptr(scal)
    a.max_norm, a.grad_scale, a.lr = max_norm, grad_scale, lr
    a.beta1, a.beta2, a.eps, a.weight_decay = betas[0], betas[1], eps, weight_decay
    if bf16_mirror is not None:
        assert bf16_mirror.dtype == torch.bfloat16 and bf16_mirror.numel() == p.numel()
        a.bf16_mirror = ptr(bf16_mirror)
    check(lib().stdiff_clip_adamw(C.byref(a), stream()))


# ---------------------------------------------------------------- norm, optimizer and 8-bit product beside the DiT
def _one_device(first, *rest):
    """Index of the device that all of these tensors are on (None entries are skipped)."""
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            require_gpu(first, t)
            raise ValueError(f"tensors on {first.device} and {t.device} in one call")
    if dev < 0:
        require_gpu(first)
    return dev


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _enqueue(dev, fn, *args):
    """check(fn(*args, stream)) with the stream that is current on device `dev`, `dev` being the current device meanwhile."""
    if dev == _current_device():
        rc = fn(*args, _current_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _current_stream(dev))
    if rc:
        check(rc)


def _lib_of(*dtypes):
    """lib_for by dtype."""
    if torch.float16 in dtypes:
        if torch.bfloat16 in dtypes:
            raise TypeError("float16 and bfloat16 tensors in one stdiff_hip call")
        return lib(True)
    return lib()


def _read_ld(t, name, shape=None):
    """Leading dimension of a matrix that is only read: rows may overlap or be one row broadcast."""
    size = t.shape
    if len(size) != 2 or (shape is not None and size != shape):
        raise ValueError(f"{name}: a matrix{'' if shape is None else f' of {tuple(shape)}'} is needed, got {tuple(size)}")
    ld, one = t.stride()
    if one != 1 and size[1] > 1:
        raise ValueError(f"{name}: the elements of a row have to be neighbours, got strides {t.stride()}")
    return ld if size[0] > 1 else size[1]


def _write_ld(t, name, shape):
    ld = _read_ld(t, name, shape)
    if ld < t.shape[1]:
        raise ValueError(f"{name}: rows of an output may not overlap, got strides {t.stride()}")
    return ld


def _vector(t, name, n, dtype=torch.float32):
    """None, or the address of a contiguous vector of n elements of this type (or of one of these)."""
    if t is None:
        return None
    kind = t.dtype
    if t.numel() != n or (t.stride() != (1,) and not (t.dim() == 1 and n <= 1)) or \
            not (kind is dtype or (dtype is _FLOATS and kind in _FLOATS)):
        raise ValueError(f"{name}: a contiguous vector of {n} elements of {dtype} is needed, got {tuple(t.shape)} {kind}")
    return t.data_ptr()


_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _affine(weight, bias, H):
    """(address, address, dtype) of a norm's weight and bias, which share one dtype."""
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype}, bias {bias.dtype}: one dtype is needed")
    one = weight if weight is not None else bias
    return _vector(weight, "weight", H, _FLOATS), _vector(bias, "bias", H, _FLOATS), torch.float32 if one is None else one.dtype


def _code(dtype):
    """The C ABI's code of a torch dtype (dt_of by dtype)."""
    if dtype is torch.float32:
        return F32
    if dtype is torch.bfloat16 or dtype is torch.float16:
        return L.BF16
    raise TypeError(f"unsupported dtype {dtype}")


def layer_norm(x, weight=None, bias=None, eps=1e-6, out=None, out_dtype=None, mean=None, rstd=None):
    """LayerNorm of the rows of x [R, H] with a weight and a bias per column (None: 1 and 0; one dtype for both).
    x and out: fp32 or a 16-bit type, any row stride, any H.  mean / rstd (fp32 [R], optional): receive the statistics
    that layer_norm_bwd takes.  out may be x."""
    dev = _one_device(x, weight, bias, out, mean, rstd)
    ldx = _read_ld(x, "x")
    R, H = x.shape
    if out is None:
        out, ldy = x.new_empty((R, H), dtype=out_dtype), H
    else:
        ldy = _write_ld(out, "out", x.shape)
    w, b, wdt = _affine(weight, bias, H)
    mp = rp = None
    if mean is not None or rstd is not None:
        mp, rp = _vector(mean, "mean", R), _vector(rstd, "rstd", R)
    xdt, ydt = x.dtype, out.dtype
    _enqueue(dev, _lib_of(xdt, ydt, wdt).stdiff_layer_norm, x.data_ptr(), ldx, _code(xdt), w, b, _code(wdt), eps, out.data_ptr(), ldy,
             _code(ydt), mp, rp, R, H)
    return out


def layer_norm_bwd(dy, x, mean, rstd, weight=None, dx=None, dweight=None, dbias=None, accumulate=False, workspace=None):
    """Backward of layer_norm from its mean / rstd: (dx, dweight, dbias).  dx has x's dtype (allocated unless given; it may be
    dy or x).  dweight / dbias are fp32 [H]: with a weight both are allocated unless given, without one those that are
    given are formed (else None); accumulate=True adds to what the given ones hold.  They are sums over the rows in a
    fixed order: the same bits every run.
    workspace (fp32, at least layer_norm_bwd_workspace(R, H, ..) floats, none for few rows; allocated unless given):
    give one of its own to a call that is captured into an ops.Graph."""
    dev = _one_device(x, dy, mean, rstd, weight, dx, dweight, dbias, workspace)
    ldx = _read_ld(x, "x")
    R, H = x.shape
    lddy = _read_ld(dy, "dy", x.shape)
    if accumulate and (dweight is None and dbias is None):
        raise ValueError("accumulate: there is no dweight or dbias to add to")
    if dx is None:
        dx, lddx = x.new_empty((R, H)), H
    elif dx.dtype != x.dtype:
        raise TypeError(f"dx is {dx.dtype}, x {x.dtype}")
    else:
        lddx = _write_ld(dx, "dx", x.shape)
    dw, db = _vector(dweight, "dweight", H), _vector(dbias, "dbias", H)
    w, wdt = None, torch.float32
    if weight is not None:
        w, wdt = _vector(weight, "weight", H, _FLOATS), weight.dtype
        if not accumulate:
            if dweight is None:
                dweight = x.new_empty((H,), dtype=torch.float32)
                dw = dweight.data_ptr()
            if dbias is None:
                dbias = x.new_empty((H,), dtype=torch.float32)
                db = dbias.data_ptr()
    if mean is None or rstd is None:
        raise ValueError("mean and rstd of the forward are needed")
    mp, rp = _vector(mean, "mean", R), _vector(rstd, "rstd", R)
    xdt, ddt = _code(x.dtype), _code(dy.dtype)
    lb = _lib_of(x.dtype, dy.dtype, wdt)
    if workspace is None and (dweight is not None or dbias is not None):
        need = lb.stdiff_layer_norm_bwd_workspace(R, H, xdt, ddt)
        if need > 0:
            workspace = x.new_empty((need // 4,), dtype=torch.float32)
    ws, nb = _workspace(workspace)
    _enqueue(dev, lb.stdiff_layer_norm_bwd, dy.data_ptr(), lddy, ddt, x.data_ptr(), ldx, xdt, mp, rp, w, _code(wdt),
             dx.data_ptr(), lddx, dw, db, int(accumulate), ws, nb, R, H)
    return dx, dweight, dbias


def layer_norm_bwd_workspace(R, H, x_dtype, dy_dtype=None):
    """Floats that layer_norm_bwd needs as workspace for x [R, H] and dy of these types (dy's is x's unless given)."""
    x_code = _code(x_dtype)
    n = lib().stdiff_layer_norm_bwd_workspace(R, H, x_code, x_code if dy_dtype is None else _code(dy_dtype))
    if n < 0:
        raise ValueError(f"layer_norm_bwd_workspace: bad size {R} x {H}")
    return n // 4


def _workspace(t):
    """(address, bytes) of a workspace tensor (None: none)."""
    if t is None:
        return None, 0
    if not t.is_contiguous():
        raise ValueError("workspace: a contiguous tensor is needed")
    return t.data_ptr(), t.numel() * t.element_size()


class AdamWTensors:
    """Parameters and their states as adamw_multi takes them (made by adamw_multi_args; holds the tensors and their memory)."""

    def __init__(self, params, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, weight_decay):
        n = len(params)
        none = [None] * n
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        lists = [list(params), list(exp_avg), list(exp_avg_sq), list(exp_avg_scale or none), list(exp_avg_sq_scale or none)]
        if any(len(t) != n for t in lists) or len(decay) != n:
            raise ValueError("adamw_multi_args: lists of different lengths")
        self.params = lists[0]
        self.state_bits = 8 if n and exp_avg[0].dtype == torch.float8_e4m3fn else 32
        kind = torch.float8_e4m3fn if self.state_bits == 8 else torch.float32
        self.table = (L.AdamWTensor * max(n, 1))()
        self.rows = np.frombuffer(self.table, dtype=np.dtype(L.AdamWTensor))[:n]
        every = [t for k in lists for t in k if t is not None]
        self.device = _one_device(*every) if n else None
        self.sizes, self.addresses = [p.numel() for p in params], [p.data_ptr() for p in params]
        for i, (p, m, v, ms, vs, size) in enumerate(zip(*lists, self.sizes)):
            if m.dtype != kind or v.dtype != kind:
                raise TypeError(f"tensor {i}: states are {m.dtype} and {v.dtype}, {kind} is needed like in the first")
            if m.numel() != size or v.numel() != size:
                raise ValueError(f"tensor {i}: states of {m.numel()} and {v.numel()} elements for {size} parameters")
            if not (p.is_contiguous() and m.is_contiguous() and v.is_contiguous()):
                raise ValueError(f"tensor {i}: the parameter or a state of it is not contiguous")
            if self.state_bits == 32 and (ms is not None or vs is not None):
                raise ValueError("32-bit states have no scales")
            if self.state_bits == 8 and (ms is None or vs is None):
                raise ValueError("8-bit states need exp_avg_scale and exp_avg_sq_scale")
            blocks = -(-size // 256)
            self.table[i] = (self.addresses[i], 0, m.data_ptr(), v.data_ptr(), _vector(ms, "exp_avg_scale", blocks),
                             _vector(vs, "exp_avg_sq_scale", blocks), size, _code(p.dtype), 0, decay[i], 0)
        ranges = sorted((t.data_ptr(), t.numel() * t.element_size()) for t in every if t.numel())
        if any(at + size > after for (at, size), (after, _) in zip(ranges, ranges[1:])):
            raise ValueError("adamw_multi_args: two of the parameters and states share memory")
        self.memory = [t.untyped_storage() for t in every]         # alive even where a tensor is given other memory
        self.partial = False                  # the last step left tensors out
        self.half = {p.dtype for p in params} - {torch.float32}
        if len(self.half) > 1:
            raise TypeError("float16 and bfloat16 parameters in one adamw_multi")


def adamw_multi_args(params, exp_avg, exp_avg_sq, exp_avg_scale=None, exp_avg_sq_scale=None, weight_decay=0.0):
    """What adamw_multi updates: lists of contiguous tensors, one entry per parameter (fp32 or one 16-bit type; views into
    larger buffers are fine).  exp_avg / exp_avg_sq: fp32, or torch.float8_e4m3fn with a vector of
    ceil(numel / 256) fp32 scales per tensor in exp_avg_scale / exp_avg_sq_scale (adamw8_state makes all four).
    weight_decay: one number, or one per tensor.  The states are read and written in place by every step."""
    return AdamWTensors(params, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, weight_decay)


def adamw8_state(param):
    """8-bit state of one parameter before its first step: (exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale), all
    zero.  exp_avg.float() * scale (of its block of 256) is the first moment, exp_avg_sq.float() * scale the ROOT of
    the second."""
    require_gpu(param)
    blocks = round_up(param.numel(), 256) // 256
    m, v = (torch.zeros(param.shape, device=param.device, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros((blocks,), device=param.device, dtype=torch.float32) for _ in range(2))
    return m, v, ms, vs


def adamw_multi_workspace(n_tensors):
    """Floats that adamw_multi needs as workspace for this many tensors."""
    n = lib().stdiff_adamw_multi_workspace(n_tensors)
    if n < 0:
        raise ValueError(f"adamw_multi_workspace: {n_tensors} tensors")
    return n // 4


def adamw_multi(args, grads, step_dev, lr, max_norm=None, grad_scale=1.0, betas=(0.9, 0.999), eps=1e-8, norm=None, workspace=None):
    """One AdamW step over all tensors of `args` (adamw_multi_args).  grads: one contiguous tensor per parameter, fp32 or a
    16-bit type, or None (that parameter and its state stay as they are).  step_dev: int32 [1] on the device, the steps
    done so far; incremented.  max_norm: clip by the norm over all gradients (None: no clipping); norm (fp32 [1],
    optional) receives that norm; grad_scale multiplies every gradient first (1 / world size, 1 / loss scale).
    workspace (fp32, at least adamw_multi_workspace(len(grads)) floats; allocated unless given): give one of its own to a
    call that is captured into an ops.Graph.  A captured step keeps lr and the other numbers it was captured with, and its
    replays do not raise the parameters' version counters: torch.autograd.graph.increment_version does."""
    sizes, rows, n = args.sizes, args.rows, len(args.sizes)
    if len(grads) != n:
        raise ValueError(f"adamw_multi: {len(grads)} gradients for {n} parameters")
    if list(map(_data_ptr, args.params)) != args.addresses:
        raise ValueError("adamw_multi: a parameter was given other memory since adamw_multi_args")
    dev = args.device if n else step_dev.get_device()
    if _one_device(step_dev, norm, workspace) != dev:
        raise ValueError(f"step_dev on {step_dev.device}, the parameters on device {dev}")
    try:
        kinds = set(map(_dtype, grads))
    except AttributeError:
        kinds = None                           # some are missing
    if kinds is not None and len(kinds) == 1:
        if args.partial:
            args.partial, rows["n"] = False, sizes
        _gradients(grads, sizes, dev, kinds, rows)
    else:
        args.partial, rows["n"] = True, 0
        kinds = set()
        for i, g in enumerate(grads):
            if g is not None:
                _gradients([g], [sizes[i]], dev, {g.dtype}, rows[i:i + 1])
                rows["n"][i] = sizes[i]
                kinds.add(g.dtype)
    kinds = (kinds | args.half) - {torch.float32}
    if len(kinds) > 1:
        raise TypeError("float16 and bfloat16 tensors in one adamw_multi")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm has to be positive (or None), got {max_norm}")
    if workspace is None:
        workspace = step_dev.new_empty((adamw_multi_workspace(n),), dtype=torch.float32)
    ws, nb = _workspace(workspace)
    a = L.AdamWMultiArgs(args.table, n, args.state_bits, _vector(step_dev, "step_dev", 1, torch.int32),
                         _vector(norm, "norm", 1), ws, nb, lr, betas[0], betas[1], eps, max_norm or 0.0, grad_scale)
    _enqueue(dev, lib(torch.float16 in kinds).stdiff_adamw_multi, C.byref(a))
    if n:
        torch.autograd.graph.increment_version(args.params)        # who keeps copies of them (DiT_stDiff) sees the change


_dtype, _numel, _get_device = operator.attrgetter("dtype"), torch.Tensor.numel, torch.Tensor.get_device
_is_contiguous, _data_ptr = torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _gradients(grads, sizes, dev, kind, rows):
    """Checks gradients of one dtype and enters them into their rows of the table."""
    if list(map(_numel, grads)) != sizes or set(map(_get_device, grads)) != {dev} or not all(map(_is_contiguous, grads)):
        raise ValueError(f"adamw_multi: contiguous gradients of the parameters' {sizes if len(sizes) < 9 else 'sizes'} elements on device "
                         f"{dev} are needed")
    rows["grad"] = list(map(_data_ptr, grads))
    for dtype in kind:
        rows["grad_dtype"] = _code(dtype)


def quantize_rows(x, out=None, scale=None):
    """(q, scale): the rows of x [R, K] (fp32 or a 16-bit type) as int8 with one fp32 scale each, scale = max |x| / 127 and
    q = rint(x * (127 / max |x|)).  q is a [R, K] view of rows that begin on 16-byte borders, zeros behind K, as gemm_i8
    takes them (a given `out` has to be such a view).  A row that holds an infinity or a NaN gets a scale that is not
    finite."""
    dev = _one_device(x, out, scale)
    ldx = _read_ld(x, "x")
    R, K = x.shape
    if out is None:
        ldq = round_up(K, 16)
        out = x.new_empty((R, ldq), dtype=torch.int8)
        if ldq != K:
            out = out[:, :K]
    else:
        ldq = _rows16(out, "out", (R, K))
    if scale is None:
        scale = x.new_empty((R,), dtype=torch.float32)
    sp = _vector(scale, "scale", R)
    _enqueue(dev, _lib_of(x.dtype).stdiff_quantize_rows, x.data_ptr(), ldx, _code(x.dtype), out.data_ptr(), ldq, sp, R, K)
    return out, scale


def _rows16(t, name, shape=None):
    """Leading dimension of an int8 matrix whose rows begin on 16-byte borders and may be touched up to the next border."""
    if t.dtype is not torch.int8:
        raise TypeError(f"{name}: int8 is needed, got {t.dtype}")
    ld = _read_ld(t, name, shape)
    rows, k = t.shape
    kp = (k + 15) & ~15
    if rows == 1:
        ld = kp
    if (ld & 15 or ld < kp or t.data_ptr() & 15 or
            (kp > k and t.storage_offset() + (rows - 1) * ld + kp > t.untyped_storage().nbytes())) and rows:
        raise ValueError(f"{name}: rows have to begin on 16-byte borders and to reach the next border behind their end in memory, "
                         f"as quantize_rows lays them out; got shape {tuple(t.shape)}, strides {t.stride()}")
    return ld


def gemm_i8(A, a_scale, W, w_scale, bias=None, out=None, out_dtype=torch.float32):
    """out[M, N] = (A[M, K] @ W[N, K]^T) * a_scale[M, None] * w_scale[N] + bias: int8 operands as quantize_rows makes them,
    the sum over K exact in int32 (K <= 131071), scales and bias fp32, out fp32 or a 16-bit type."""
    dev = _one_device(A, a_scale, W, w_scale, bias, out)
    lda, ldw = _rows16(A, "A"), _rows16(W, "W")
    (M, K), N = A.shape, W.shape[0]
    if W.shape[1] != K:
        raise ValueError(f"A has {K} columns, W {W.shape[1]}")
    if a_scale is None or w_scale is None:
        raise ValueError("a_scale and w_scale are needed")
    if out is None:
        out, ldc = a_scale.new_empty((M, N), dtype=out_dtype), N
    else:
        ldc = _write_ld(out, "out", (M, N))
    a = L.GemmI8Args(M, N, K, A.data_ptr(), lda, W.data_ptr(), ldw, _vector(a_scale, "a_scale", M),
                     _vector(w_scale, "w_scale", N), _vector(bias, "bias", N), out.data_ptr(), ldc,
                     _code(out.dtype))
    _enqueue(dev, _lib_of(out.dtype).stdiff_gemm_i8, C.byref(a))
    return out


class Graph:
    """hipGraph capture of everything enqueued on the current stream between begin() and end()."""

    def __init__(self):
        self.exec = None

    def begin(self):
        check(lib().stdiff_graph_begin(stream()))

    def end(self):
        h = C.c_void_p()
        check(lib().stdiff_graph_end(stream(), C.byref(h)))
        self.exec = h

    def launch(self):
        check(lib().stdiff_graph_launch(self.exec, stream()))

    def __del__(self):
        if self.exec is not None:
            try:
                lib().stdiff_graph_destroy(self.exec)
            except Exception:
                pass
            self.exec = None
