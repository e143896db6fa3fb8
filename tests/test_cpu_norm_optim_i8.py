"""CPU: what the entry points of the layer norm, AdamW and 8-bit product refuse before they launch anything (through the C
ABI with addresses that are never read), their workspace sizes, their structs, and the checks of the Python layer."""
import ctypes as C
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -6
AT = 1 << 20                                            # an aligned address that nothing lies at


@pytest.fixture(scope="module", params=[False, True], ids=["bf16", "fp16"])
def lib(request):
    from stdiff_amd import _lib
    return _lib.lib(request.param)


def test_layer_norm_refuses(lib):
    def fwd(x=AT, ldx=64, xd=0, w=AT, b=AT, wd=0, eps=1e-6, y=AT, ldy=64, yd=0, mean=None, rstd=None, R=4, H=64):
        return lib.stdiff_layer_norm(x, ldx, xd, w, b, wd, eps, y, ldy, yd, mean, rstd, R, H, None)
    for kw in (dict(x=None), dict(y=None), dict(R=-1), dict(H=0), dict(ldx=-1), dict(ldy=63), dict(eps=-1.0), dict(eps=float("nan")),
               dict(xd=2), dict(yd=-1), dict(wd=7)):
        assert fwd(**kw) == ARG, kw
    for kw in (dict(x=AT + 2), dict(y=AT + 1, yd=1), dict(w=AT + 3), dict(mean=AT + 2), dict(rstd=AT + 1)):
        assert fwd(**kw) == ALIGN, kw
    assert fwd(R=0, x=None, y=None) == 0


def test_layer_norm_bwd_refuses(lib):
    need = lib.stdiff_layer_norm_bwd_workspace(9000, 1001, 0, 0)
    for bad in ((-1, 5, 0, 0), (5, 0, 0, 0), (5, 5, 2, 0), (5, 5, 1, -1)):
        assert lib.stdiff_layer_norm_bwd_workspace(*bad) == ARG
    assert need > 0 and lib.stdiff_layer_norm_bwd_workspace(0, 5, 1, 1) >= 0 and lib.stdiff_layer_norm_bwd_workspace(10, 5, 0, 1) >= 0

    def bwd(dy=AT, ldd=1001, dd=0, x=AT, ldx=1001, xd=0, mean=AT, rstd=AT, w=AT, wd=0, dx=AT, lddx=1001, dw=AT, db=AT, ws=AT, nb=need, R=9000, H=1001):
        return lib.stdiff_layer_norm_bwd(dy, ldd, dd, x, ldx, xd, mean, rstd, w, wd, dx, lddx, dw, db, 0, ws, nb, R, H, None)
    for kw in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(dx=None), dict(lddx=1000), dict(ldd=-1), dict(R=-2), dict(H=-1),
               dict(dd=2), dict(xd=3), dict(wd=-1)):
        assert bwd(**kw) == ARG, kw
    for kw in (dict(dy=AT + 1), dict(dx=AT + 2), dict(dw=AT + 2), dict(ws=AT + 4)):
        assert bwd(**kw) == ALIGN, kw
    for kw in (dict(ws=None), dict(nb=need - 1), dict(nb=0), dict(db=None, nb=0)):
        assert bwd(**kw) == WORKSPACE, kw
    assert bwd(R=0, dw=None, db=None, ws=None, nb=0, dy=None, x=None, dx=None, mean=None, rstd=None) == 0


def test_adamw_multi_refuses(lib):
    from stdiff_amd import _lib as L
    need = lib.stdiff_adamw_multi_workspace(2)
    assert need > 0 and lib.stdiff_adamw_multi_workspace(-1) == ARG
    assert lib.stdiff_adamw_multi_workspace(500) > need

    def step(bits=32, n=2, change=None, **kw):
        t = (L.AdamWTensor * 2)()
        for q in t:
            q.param = q.grad = q.exp_avg = q.exp_avg_sq = q.exp_avg_scale = q.exp_avg_sq_scale = AT
            q.n = 1000
        for k, v in (change or {}).items():
            setattr(t[1], k, v)
        a = L.AdamWMultiArgs()
        a.tensors, a.n_tensors, a.state_bits = t, n, bits
        a.step_dev, a.workspace, a.workspace_bytes = AT, AT, need
        a.lr, a.beta1, a.beta2, a.eps, a.max_norm, a.grad_scale = 1e-3, 0.9, 0.999, 1e-8, 1.0, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.stdiff_adamw_multi(C.byref(a), None)
    assert lib.stdiff_adamw_multi(None, None) == ARG
    for kw in (dict(bits=16), dict(n=-1), dict(step_dev=None), dict(workspace=None), dict(beta1=1.0), dict(beta2=-0.1), dict(beta1=float("nan")),
               dict(eps=-1e-8), dict(lr=-1.0), dict(lr=float("nan")), dict(max_norm=float("nan"))):
        assert step(**kw) == ARG, kw
    for ch in (dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(n=-1), dict(param_dtype=2), dict(grad_dtype=9)):
        assert step(change=ch) == ARG, ch
    for ch in (dict(exp_avg_scale=None), dict(exp_avg_sq_scale=None)):
        assert step(bits=8, change=ch) == ARG, ch
    for ch in (dict(param=AT + 2), dict(grad=AT + 1), dict(exp_avg=AT + 2)):
        assert step(change=ch) == ALIGN, ch
    assert step(bits=8, change=dict(exp_avg_sq_scale=AT + 2)) == ALIGN
    assert step(workspace_bytes=need - 1) == WORKSPACE
    assert step(change=dict(n=1 << 45)) == SHAPE


def test_product_refuses(lib):
    from stdiff_amd import _lib as L

    def prod(**kw):
        a = L.GemmI8Args()
        a.M, a.N, a.K = 10, 20, 100
        a.A = a.W = a.a_scale = a.w_scale = a.bias = a.C = AT
        a.lda = a.ldw = 112
        a.ldc = 20
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.stdiff_gemm_i8(C.byref(a), None)
    assert lib.stdiff_gemm_i8(None, None) == ARG
    for kw in (dict(A=None), dict(W=None), dict(a_scale=None), dict(w_scale=None), dict(C=None), dict(M=-1), dict(N=-5), dict(K=0), dict(lda=96),
               dict(ldw=96), dict(ldc=19), dict(c_dtype=2)):
        assert prod(**kw) == ARG, kw
    for kw in (dict(lda=120), dict(ldw=113), dict(A=AT + 8), dict(W=AT + 1), dict(C=AT + 2), dict(bias=AT + 2), dict(a_scale=AT + 1)):
        assert prod(**kw) == ALIGN, kw
    assert prod(K=131072, lda=131072, ldw=131072) == SHAPE and prod(lda=1 << 24) == SHAPE
    assert prod(M=0, A=None, C=None) == 0 and prod(N=0) == 0

    def quant(x=AT, ldx=100, xd=0, q=AT, ldq=112, s=AT, R=3, K=100):
        return lib.stdiff_quantize_rows(x, ldx, xd, q, ldq, s, R, K, None)
    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(R=-1), dict(K=0), dict(ldx=-1), dict(ldq=100), dict(ldq=96), dict(xd=2)):
        assert quant(**kw) == ARG, kw
    for kw in (dict(ldq=120), dict(q=AT + 8), dict(x=AT + 2), dict(s=AT + 2)):
        assert quant(**kw) == ALIGN, kw
    assert quant(R=0, x=None, q=None, s=None) == 0


def test_structs_match_the_header(tmp_path):
    """sizes and offsets of the new structs as a C compiler lays them out"""
    import subprocess
    from stdiff_amd import _lib as L
    pairs = (("stdiff_adamw_tensor", L.AdamWTensor), ("stdiff_adamw_multi_args", L.AdamWMultiArgs), ("stdiff_gemm_i8_args", L.GemmI8Args))
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "stdiff_hip.h"', 'int main(void) {']
    for name, cls in pairs:
        src.append(f'printf("%zu\\n", sizeof({name}));')
        src += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    (tmp_path / "t.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def test_tensors_are_checked_first():
    """what is wrong with the tensors themselves is refused without a GPU too, with the argument's name"""
    from stdiff_amd import ops
    x, w, s4 = torch.zeros(4, 32), torch.ones(32), torch.zeros(4)

    def refused(kind, match, call):
        with pytest.raises(kind, match=match):
            call()
    for bad in (x.t(), x[:, ::2], x[0], x[None]):
        refused(ValueError, "x:", lambda: ops.layer_norm(bad))
    for bad in (torch.ones(31), torch.ones(64)[::2], torch.ones(32, 1), torch.ones(32).double(), torch.ones(32).int()):
        refused(ValueError, "weight:", lambda: ops.layer_norm(x, bad))
    refused(TypeError, "one dtype", lambda: ops.layer_norm(x, w, w.bfloat16()))
    refused(TypeError, "float16 and bfloat16", lambda: ops.layer_norm(x.half(), w.bfloat16()))
    refused(TypeError, "dtype", lambda: ops.layer_norm(x.double()))
    refused(TypeError, "dtype", lambda: ops.layer_norm(x, out_dtype=torch.int32))
    refused(TypeError, "tensor", lambda: ops.layer_norm([1.0]))
    refused(TypeError, "torch.dtype", lambda: ops.layer_norm(x, out_dtype="fp32"))
    refused(TypeError, "real number", lambda: ops.layer_norm(x, eps="small"))
    refused(ValueError, "overlap", lambda: ops.layer_norm(x, out=torch.zeros(32).expand(4, 32)))
    refused(ValueError, "out:", lambda: ops.layer_norm(x, out=torch.zeros(4, 31)))
    refused(ValueError, "mean", lambda: ops.layer_norm(x, mean=torch.zeros(5)))
    refused(ValueError, "mean and rstd", lambda: ops.layer_norm_bwd(x, x, s4, None))
    refused(ValueError, "dy:", lambda: ops.layer_norm_bwd(x[:3], x, s4, s4))
    refused(ValueError, "accumulate", lambda: ops.layer_norm_bwd(x, x, s4, s4, w, accumulate=True))
    refused(ValueError, "dweight", lambda: ops.layer_norm_bwd(x, x, s4, s4, w, dweight=w.bfloat16()))
    refused(TypeError, "dx is", lambda: ops.layer_norm_bwd(x, x, s4, s4, w, dx=x.bfloat16()))
    refused(ValueError, "workspace", lambda: ops.layer_norm_bwd(x, x, s4, s4, w, workspace=torch.zeros(8, 8).t()))
    q = torch.zeros(5, 48, dtype=torch.int8)
    assert q.data_ptr() % 16 == 0
    ones = torch.ones(5)
    for bad in (q[:, 1:20], torch.zeros(5, 40, dtype=torch.int8), torch.zeros(4 * 48 + 40, dtype=torch.int8).as_strided((5, 40), (48, 1))):
        refused(ValueError, "A: rows", lambda: ops.gemm_i8(bad, ones, q, ones))
        refused(ValueError, "out: rows", lambda: ops.quantize_rows(torch.zeros(bad.shape), out=bad))
    for good in (q, q[:, :40], q[:1, :3], q[4:, 32:40]):
        n = torch.ones(good.shape[0])
        refused(RuntimeError, "MI355X", lambda: ops.gemm_i8(good, n, good, n))
    refused(TypeError, "W: int8", lambda: ops.gemm_i8(q, ones, q.float(), ones))
    refused(ValueError, "columns", lambda: ops.gemm_i8(q, ones, q[:, :16], ones))
    refused(ValueError, "w_scale", lambda: ops.gemm_i8(q, ones, q, torch.ones(4)))
    refused(ValueError, "are needed", lambda: ops.gemm_i8(q, None, q, ones))
    refused(ValueError, "out:", lambda: ops.gemm_i8(q, ones, q, ones, out=torch.zeros(5, 6)))
    p, m, v = (torch.zeros(300) for _ in range(3))
    refused(ValueError, "lengths", lambda: ops.adamw_multi_args([p], [m], []))
    refused(ValueError, "lengths", lambda: ops.adamw_multi_args([p], [m], [v], weight_decay=[0.0, 1.0]))
    refused(TypeError, "states are", lambda: ops.adamw_multi_args([p], [m.half()], [v]))
    refused(ValueError, "states of", lambda: ops.adamw_multi_args([p], [m[:7]], [v]))
    refused(ValueError, "contiguous", lambda: ops.adamw_multi_args([torch.zeros(600)[::2]], [m], [v]))
    refused(ValueError, "scales", lambda: ops.adamw_multi_args([p], [m], [v], [ones], [ones]))
    refused(TypeError, "float16 and bfloat16", lambda: ops.adamw_multi_args([p.half(), p.bfloat16()], [m, m.clone()], [v, v.clone()]))
    c = [torch.zeros(300).to(torch.float8_e4m3fn) for _ in range(2)]
    refused(ValueError, "8-bit", lambda: ops.adamw_multi_args([p], c[:1], c[1:]))
    refused(ValueError, "exp_avg_scale", lambda: ops.adamw_multi_args([p], c[:1], c[1:], [torch.zeros(1)], [torch.zeros(2)]))


def test_no_cpu_path():
    from stdiff_amd import ops
    x, q, s = torch.zeros(4, 16), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    p = torch.zeros(8)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_bwd(x, x, s, s), lambda: ops.quantize_rows(x), lambda: ops.gemm_i8(q, s, q, s),
                 lambda: ops.adamw_multi_args([p], [p], [p]), lambda: ops.adamw8_state(p)):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_longest_rows_and_decay(lib):
    """columns are counted in 32 bits with a workgroup's stride behind them; a weight decay is not negative"""
    from stdiff_amd import _lib as L
    H = (1 << 30) + 1
    assert lib.stdiff_layer_norm(AT, H, 0, AT, AT, 0, 1e-6, AT, H, 0, None, None, 1, H, None) == SHAPE
    assert lib.stdiff_layer_norm(AT, 2**31 - 1, 1, None, None, 0, 1e-6, AT, 2**31 - 1, 1, None, None, 3, 2**31 - 1, None) == SHAPE
    assert lib.stdiff_layer_norm_bwd_workspace(4, H, 0, 0) == SHAPE
    assert lib.stdiff_layer_norm_bwd(AT, H, 0, AT, H, 0, AT, AT, AT, 0, AT, H, AT, AT, 0, AT, 1 << 50, 4, H, None) == SHAPE
    for wd in (-0.1, float("nan")):
        t = (L.AdamWTensor * 1)()
        t[0].param = t[0].grad = t[0].exp_avg = t[0].exp_avg_sq = AT
        t[0].n, t[0].weight_decay = 5, wd
        a = L.AdamWMultiArgs()
        a.tensors, a.n_tensors, a.state_bits = t, 1, 32
        a.step_dev, a.workspace, a.workspace_bytes = AT, AT, 1 << 20
        a.lr, a.beta1, a.beta2, a.eps, a.grad_scale = 1e-3, 0.9, 0.999, 1e-8, 1.0
        assert lib.stdiff_adamw_multi(C.byref(a), None) == ARG, wd


def test_shared_memory_is_refused():
    """an output may be the input where that is said, and may lie beside it in one buffer; everything else that overlaps is refused"""
    from stdiff_amd import ops
    buf, s4, w = torch.zeros(4, 96), torch.zeros(4), torch.ones(32)
    x = buf[:, 32:64]

    def refused(match, call, kind=ValueError):
        with pytest.raises(kind, match=match):
            call()
    for out in (buf[:, 31:63], buf[:, 33:65], buf.view(-1)[32:160].view(4, 32)):
        refused("share memory", lambda: ops.layer_norm(x, out=out))
        refused("share memory", lambda: ops.layer_norm_bwd(torch.zeros(4, 32), x, s4, s4, dx=out))
        refused("share memory", lambda: ops.layer_norm_bwd(x, torch.zeros(4, 32), s4, s4, dx=out))
    refused("share memory", lambda: ops.layer_norm(x, out=buf.view(torch.bfloat16)[:, 64:96]))
    refused("share memory", lambda: ops.layer_norm(buf[:1, :32].expand(4, 32), out=buf[:, :32]))
    # the same elements, columns beside them, the other rows: these are fine as far as a machine without a GPU can tell
    for out in (x, buf[:, :32], buf[:, 64:], torch.zeros(4, 32)):
        refused("MI355X", lambda: ops.layer_norm(x, out=out), RuntimeError)
        refused("MI355X", lambda: ops.layer_norm_bwd(x, x, s4, s4, dx=out), RuntimeError)
    rows = torch.zeros(8, 32)
    refused("MI355X", lambda: ops.layer_norm(rows[:4], out=rows[4:]), RuntimeError)
    refused("share memory", lambda: ops.layer_norm(rows[:4], out=rows[3:7]))
    refused("MI355X", lambda: ops.layer_norm(rows[::2], out=rows[1::2]), RuntimeError)
    refused("mean and rstd", lambda: ops.layer_norm(x, mean=s4, rstd=s4))
    refused("dweight and dbias", lambda: ops.layer_norm_bwd(x, x, s4, s4, w, dweight=w, dbias=w))
    refused("share memory", lambda: ops.quantize_rows(buf, out=buf.view(torch.int8)[:, :96]))
    q = torch.zeros(4, 32, dtype=torch.int8)
    refused("out and A", lambda: ops.gemm_i8(q, s4, q.clone(), s4, out=q.view(torch.float32)[:, :4]))
    refused("out and W", lambda: ops.gemm_i8(q.clone(), s4, q, s4, out=q.view(torch.float32)[:, :4]))


def test_without_the_extension_module(tmp_path):
    """what does not need _bind works without it, what needs it says what is missing"""
    import subprocess
    import sys
    code = ("import sys; sys.modules['stdiff_amd._bind'] = None\n"
            "import torch; from stdiff_amd import ops\n"
            "assert ops.round_up(5, 4) == 8 and ops.adamw_multi_workspace(1) > 0\n"
            "try: ops.layer_norm(torch.zeros(2, 8))\n"
            "except RuntimeError as e: print('refused', e)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and "refused stdiff_amd/_bind.so cannot be used" in r.stdout, r.stderr


def test_largest_products(lib):
    """rows and columns of C are counted in 32 bits with a tile behind them: more than 2^30 of either are refused"""
    from stdiff_amd import _lib as L
    for M, N in (((1 << 30) + 1, 8), (8, (1 << 30) + 1), (2**31 - 1, 1), (1, 2**31 - 1)):
        a = L.GemmI8Args()
        a.M, a.N, a.K = M, N, 16
        a.A = a.W = a.a_scale = a.w_scale = a.C = AT
        a.lda = a.ldw = 16
        a.ldc = N
        for c_dtype in (0, 1):
            a.c_dtype = c_dtype
            assert lib.stdiff_gemm_i8(C.byref(a), None) == SHAPE, (M, N, c_dtype)


def test_quantize_rows_padding_is_kept_apart():
    """the rows of q are written up to the next 16-byte border, so x may lie behind that, not behind K"""
    from stdiff_amd import ops
    buf = torch.zeros(4, 64)
    q = buf.view(torch.int8)
    assert q.data_ptr() % 16 == 0
    for rows in (4, 1):
        for first in (10, 11):                                # bytes 40 and 44 of the row, q's end at 48
            with pytest.raises(ValueError, match="out and x share memory"):
                ops.quantize_rows(buf[:rows, first:first + 40], out=q[:rows, :40])
        with pytest.raises(ValueError, match="out and x share memory"):
            ops.quantize_rows(buf.view(torch.bfloat16)[:rows, 3:8], out=q[:rows, :5])      # in the padding alone
        with pytest.raises(RuntimeError, match="MI355X"):
            ops.quantize_rows(buf[:rows, 12:52], out=q[:rows, :40])
        with pytest.raises(RuntimeError, match="MI355X"):
            ops.quantize_rows(buf[:rows, :40], out=q[:rows, 160:200])


def apart(call):
    """as far as a machine without a GPU can tell, the call's tensors may lie where they do"""
    with pytest.raises(RuntimeError, match="MI355X"):
        call()


def shared(names, call):
    with pytest.raises(ValueError, match=f"{names} share memory"):
        call()


def test_layer_norm_outputs_are_kept_apart():
    """out, mean and rstd against everything that is read, and against each other; in the gaps between rows they may lie"""
    from stdiff_amd import ops
    buf = torch.zeros(8, 64)
    x, w, b, flat = buf[:4, :32], torch.ones(32), torch.zeros(32), buf.view(-1)
    shared("out and weight", lambda: ops.layer_norm(x, buf[5, :32], out=buf[4:, :32]))
    shared("out and bias", lambda: ops.layer_norm(x, w, buf[7, 31:63], out=buf[4:, :32]))
    shared("out and weight", lambda: ops.layer_norm(x, x[2], out=x))
    shared("out and mean", lambda: ops.layer_norm(x, mean=buf[6, 29:33], out=buf[4:, :32]))
    shared("out and rstd", lambda: ops.layer_norm(x, rstd=flat[4 * 64 - 3:4 * 64 + 1], out=buf[4:, :32]))
    shared("mean and x", lambda: ops.layer_norm(x, mean=buf[3, 28:32]))
    shared("rstd and x", lambda: ops.layer_norm(x, rstd=buf[0, :4]))
    shared("mean and weight", lambda: ops.layer_norm(x, w, mean=w[:4]))
    shared("rstd and weight", lambda: ops.layer_norm(x, w, rstd=w[28:]))
    shared("mean and bias", lambda: ops.layer_norm(x, w, b, mean=b[5:9]))
    shared("rstd and bias", lambda: ops.layer_norm(x, w, b, rstd=b[:4]))
    shared("mean and rstd", lambda: ops.layer_norm(x, mean=w[:4], rstd=w[3:7]))
    for at in (buf[0, 32:], buf[3, 32:], buf[2, 32:], flat[4 * 64:4 * 64 + 32]):
        apart(lambda: ops.layer_norm(x, at[:32], at[:32], mean=flat[6 * 64:6 * 64 + 4], rstd=flat[7 * 64:7 * 64 + 4], out=x))
    apart(lambda: ops.layer_norm(x, w, w, mean=buf[1, 32:36], rstd=buf[1, 36:40], out=buf[4:, 32:]))
    # a row of its own as weight: of another row nothing is written
    apart(lambda: ops.layer_norm(buf[:1, :32], buf[1, :32], buf[2, :32], out=buf[:1, :32]))
    apart(lambda: ops.layer_norm(torch.zeros(0, 32), w, w, out=torch.zeros(0, 32), mean=w[:0], rstd=w[:0]))


def test_layer_norm_bwd_outputs_are_kept_apart():
    """dx, dweight, dbias and a given workspace against everything that is read, and against each other"""
    from stdiff_amd import ops
    buf = torch.zeros(12, 64)
    x, dy, flat = buf[:4, :32], buf[4:8, :32], buf.view(-1)
    w, s1, s2, g1, g2 = torch.ones(32), torch.zeros(4), torch.zeros(4), torch.zeros(32), torch.zeros(32)
    ws = torch.zeros(4096)

    def bwd(dy=dy, x=x, mean=s1, rstd=s2, w=w, **kw):
        return lambda: ops.layer_norm_bwd(dy, x, mean, rstd, w, **kw)
    assert ops.layer_norm_bwd_workspace(4, 32, torch.float32) == 0
    shared("dweight and weight", bwd(dweight=w))
    shared("dbias and weight", bwd(dbias=w))
    shared("dweight and x", bwd(dweight=buf[3, :32]))
    shared("dbias and dy", bwd(dbias=buf[4, 20:52]))
    shared("dweight and mean", bwd(mean=g1[3:7], dweight=g1))
    shared("dbias and rstd", bwd(rstd=g2[28:], dbias=g2))
    shared("dx and weight", bwd(w=buf[8, :32], dx=buf[8:, :32]))
    shared("dx and mean", bwd(mean=buf[11, 28:32], dx=buf[8:, :32]))
    shared("dx and rstd", bwd(rstd=buf[9, 31:35], dx=buf[8:, :32]))
    shared("dx and dweight", bwd(dweight=buf[10, 16:48], dx=buf[8:, :32]))
    shared("dx and dbias", bwd(dbias=x[0], dx=x))
    shared("dweight and dbias", bwd(dweight=ws[:32], dbias=ws[31:63]))
    for name, kw in (("x", {}), ("dy", {}), ("dx", dict(dx=buf[8:, :32])), ("weight", {}), ("mean", {}), ("rstd", {}), ("dweight", dict(dweight=g1)),
                     ("dbias", dict(dbias=g2))):
        over = {"x": flat[200:260], "dy": flat[4 * 64 + 31:4 * 64 + 33], "dx": flat[8 * 64:8 * 64 + 4], "weight": w, "mean": s1, "rstd": s2[1:],
                "dweight": g1[:16], "dbias": g2[16:]}[name]
        shared(f"workspace and {name}", bwd(workspace=over, **kw))
    for dx in (x, dy, buf[8:, :32], buf[:4, 32:]):
        apart(bwd(dx=dx, dweight=g1, dbias=g2, workspace=ws))
    apart(bwd(w=buf[1, 32:], mean=buf[2, 32:36], rstd=buf[2, 36:40], dweight=buf[3, 32:], dbias=buf[5, 32:], dx=x, workspace=flat[8 * 64:]))
    apart(bwd(dy=dy[:1].expand(4, 32), dweight=dy[1], dbias=dy[2], dx=x))


def test_quantize_rows_scale_is_kept_apart():
    """scale against x and out, the padding of out's rows included"""
    from stdiff_amd import ops
    buf = torch.zeros(8, 64)
    x, q = buf[:4, :32], buf.view(torch.int8)[4:, :40]
    assert q.data_ptr() % 16 == 0
    shared("scale and x", lambda: ops.quantize_rows(x, scale=buf[3, 28:32]))
    shared("scale and x", lambda: ops.quantize_rows(x[:1].expand(4, 32), scale=buf[0, :4]))
    shared("out and scale", lambda: ops.quantize_rows(buf[:4, :40], out=q, scale=buf[5, 9:13]))
    shared("out and scale", lambda: ops.quantize_rows(buf[:4, :40], out=q, scale=buf[5, 11:15]))      # in the padding: bytes 44 to 47
    shared("out and scale", lambda: ops.quantize_rows(buf[:4, :40], out=q, scale=buf.view(-1)[4 * 64 - 1:4 * 64 + 3]))
    for scale in (buf[5, 12:16], buf[0, 40:44], torch.zeros(4)):
        apart(lambda: ops.quantize_rows(buf[:4, :40], out=q, scale=scale))


def test_gemm_i8_output_is_kept_apart():
    """out against the scales and the bias; in the gaps between its rows they may lie"""
    from stdiff_amd import ops
    A, W = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(6, 32, dtype=torch.int8)
    sa, sw, b, buf = torch.ones(4), torch.ones(6), torch.zeros(6), torch.zeros(4, 16)
    out = buf[:, :6]
    shared("out and bias", lambda: ops.gemm_i8(A, sa, W, sw, buf[2, :6], out=out))
    shared("out and bias", lambda: ops.gemm_i8(A, sa, W, sw, buf[2, 5:11], out=out))
    shared("out and a_scale", lambda: ops.gemm_i8(A, buf[0, 4:8], W, sw, b, out=out))
    shared("out and w_scale", lambda: ops.gemm_i8(A, sa, W, buf.view(-1)[11:17], b, out=out))
    shared("out and w_scale", lambda: ops.gemm_i8(A, sa, W, buf[3, :6], b, out=buf.view(torch.bfloat16)[:, 10:16]))
    apart(lambda: ops.gemm_i8(A, buf[0, 6:10], W, buf[1, 6:12], buf[2, 10:16], out=out))
    apart(lambda: ops.gemm_i8(A, sa, W, sw, sw, out=out))


def test_workspace_queries_refuse_what_an_int_cannot_hold():
    """sizes reach the C ABI as they are given, or are refused; they do not wrap"""
    from stdiff_amd import ops
    for n in (-1, 5 - 2**32, 2**31, 2**32 + 1, 2**64 + 1):
        with pytest.raises(ValueError):
            ops.adamw_multi_workspace(n)
        with pytest.raises(ValueError):
            ops.layer_norm_bwd_workspace(n, 64, torch.float32)
        with pytest.raises(ValueError):
            ops.layer_norm_bwd_workspace(64, n, torch.float32)
    assert ops.layer_norm_bwd_workspace(2**31 - 1, 64, torch.float32) > 0 and ops.adamw_multi_workspace(2**31 - 1) > 2**31


def test_build_compiles_what_is_built_already(monkeypatch):
    """build() leaves no object of older sources or flags in place, whatever its time stamp says"""
    import __graft_entry__ as G
    ran = []
    monkeypatch.setattr(G.subprocess, "run", lambda cmd, **kw: ran.append(cmd))
    G.build()
    assert len(ran) == 2 and all(cmd[0] == "make" and "-B" in cmd for cmd in ran)
