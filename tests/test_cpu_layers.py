"""Refusals of the layer operators, on the CPU: the C entry points look at sizes, strides, pointers and workspaces before any
launch, the Python ones at types, shapes and devices.  Nothing here launches a kernel."""
import ctypes

import pytest
import torch

from nerf_loc_amd import helpers, hip, layers

P = ctypes.c_void_p(4096)        # a pointer that no refused call may follow
INVALID = -1


def linear(lib, dt=0, x0=P, ldx0=8, k0=8, x1=None, ldx1=0, k1=0, w=P, ldw=8, bias=None, act=0, res=None, ldr=0, y=P, ldy=4, z=None,
           ldz=0, M=2, N=4, ws=None, nws=0):
    return lib.nerf_linear(dt, x0, ldx0, k0, x1, ldx1, k1, w, ldw, bias, act, res, ldr, y, ldy, z, ldz, M, N, ws, nws, None)


@pytest.mark.parametrize("bad", [dict(dt=3), dict(dt=-1), dict(act=4), dict(act=-1), dict(M=-1), dict(M=1 << 31), dict(N=0), dict(k0=0),
                                 dict(k1=-1), dict(k0=(1 << 24) + 1), dict(x0=None), dict(w=None), dict(y=None), dict(k1=2, ldw=10),
                                 dict(ldx0=7), dict(ldw=7), dict(ldy=3), dict(res=P, ldr=3), dict(z=P, ldz=3),
                                 dict(k1=2, x1=P, ldx1=1, ldw=10), dict(k1=2, x1=P, ldx1=2, ldw=9)], ids=str)
def test_linear_refuses(bad):
    lib = hip.lib()
    assert linear(lib, **bad) == INVALID
    assert lib.nerf_last_error()


def test_linear_refuses_a_short_or_unaligned_workspace():
    lib = hip.lib()
    # 4096 rows of 1021 through 1024 outputs: copied first
    need = lib.nerf_linear_workspace_bytes(1, P, 1021, 1021, None, 0, 0, P, 1021, 4096, 1024)
    assert need > 4096 * 1024 * 2
    big = dict(dt=1, ldx0=1021, k0=1021, ldw=1021, ldy=1024, M=4096, N=1024)
    assert linear(lib, **big) == INVALID
    assert linear(lib, **big, ws=P, nws=need - 1) == INVALID and b"workspace" in lib.nerf_last_error()
    assert linear(lib, **big, ws=ctypes.c_void_p(4096 + 16), nws=need) == INVALID and b"256" in lib.nerf_last_error()
    # aligned rows and few rows take none, whatever the size
    assert lib.nerf_linear_workspace_bytes(1, P, 1024, 1024, None, 0, 0, P, 1024, 65536, 1024) == 0
    assert lib.nerf_linear_workspace_bytes(1, P, 1021, 1021, None, 0, 0, P, 1021, 64, 1024) == 0
    # sizes that the call would refuse need nothing
    assert lib.nerf_linear_workspace_bytes(7, P, 8, 8, None, 0, 0, P, 8, 2, 4) == 0
    assert lib.nerf_linear_workspace_bytes(0, P, 8, 8, None, 0, 0, P, 8, -2, 4) == 0


def test_no_rows_need_no_pointers():
    lib = hip.lib()
    assert linear(lib, M=0, x0=None, w=None, y=None) == 0
    assert lib.nerf_linear_q8(None, 8, None, None, 8, None, 1, None, 0, None, 0, None, 4, 0, 4, 8, None, 0, None) == 0
    assert lib.nerf_add_rms_norm(0, None, 8, None, 0, None, 1e-6, None, 0, None, 8, None, 0, None, None, 0, 8, None) == 0


def backward(lib, dt=0, g=P, ldg=4, z=None, ldz=0, act=0, x0=P, ldx0=8, k0=8, x1=None, ldx1=0, k1=0, w=P, ldw=8, dx0=P, lddx0=8,
             dx1=None, lddx1=0, dw=P, db=P, M=2, N=4, ws=P, nws=1 << 30):
    return lib.nerf_linear_backward(dt, g, ldg, z, ldz, act, x0, ldx0, k0, x1, ldx1, k1, w, ldw, dx0, lddx0, dx1, lddx1, dw, db, M, N,
                                    ws, nws, None)


@pytest.mark.parametrize("bad", [dict(dt=9), dict(act=9), dict(M=-1), dict(N=0), dict(g=None), dict(act=1), dict(act=1, z=P, ldz=3),
                                 dict(x0=None), dict(w=None), dict(dx1=P, lddx1=8), dict(ldg=3), dict(ldx0=7), dict(ldw=7),
                                 dict(lddx0=7), dict(ws=None, nws=0), dict(ws=ctypes.c_void_p(4096 + 8))], ids=str)
def test_linear_backward_refuses(bad):
    assert backward(hip.lib(), **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(out=3), dict(act=7), dict(M=-1), dict(N=0), dict(K=0), dict(xq=None), dict(xs=None), dict(wq=None),
                                 dict(ws=None), dict(y=None), dict(ldx=7), dict(ldw=7), dict(ldy=3), dict(res=P, ldr=3)], ids=str)
def test_linear_q8_refuses(bad):
    a = dict(xq=P, ldx=8, xs=P, wq=P, ldw=8, ws=P, out=1, bias=None, act=0, res=None, ldr=0, y=P, ldy=4, M=2, N=4, K=8)
    a.update(bad)
    assert hip.lib().nerf_linear_q8(a["xq"], a["ldx"], a["xs"], a["wq"], a["ldw"], a["ws"], a["out"], a["bias"], a["act"], a["res"],
                                    a["ldr"], a["y"], a["ldy"], a["M"], a["N"], a["K"], None, 0, None) == INVALID


@pytest.mark.parametrize("bad", [dict(dt=5), dict(M=-1), dict(N=0), dict(N=32769, ld=32769), dict(x=None), dict(w=None), dict(y=None),
                                 dict(q=P), dict(y=None, q=P), dict(ld=7), dict(eps=-1.0), dict(eps=float("nan"))], ids=str)
def test_add_rms_norm_refuses(bad):
    a = dict(dt=0, x=P, ld=8, w=P, eps=1e-6, y=P, q=None, scale=None, M=2, N=8)
    a.update(bad)
    assert hip.lib().nerf_add_rms_norm(a["dt"], a["x"], a["ld"], None, 0, a["w"], a["eps"], None, 0, a["y"], a["ld"], a["q"], a["ld"],
                                       a["scale"], None, a["M"], a["N"], None) == INVALID


@pytest.mark.parametrize("bad", [dict(dt=5), dict(M=-1), dict(N=40000), dict(gy=None), dict(h=None), dict(w=None), dict(rstd=None),
                                 dict(dx=None, dw=None), dict(ld=7), dict(nws=0)], ids=str)
def test_add_rms_norm_backward_refuses(bad):
    a = dict(dt=0, gy=P, ld=8, h=P, w=P, rstd=P, dx=P, dw=P, M=2000, N=8, nws=1 << 20)
    a.update(bad)
    assert hip.lib().nerf_add_rms_norm_backward(a["dt"], a["gy"], a["ld"], None, 0, a["h"], a["ld"], a["w"], a["rstd"], a["dx"], a["ld"],
                                                a["dw"], a["M"], a["N"], P, a["nws"], None) == INVALID


def test_python_entries_refuse():
    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    for call in (lambda: layers.linear(x, w), lambda: layers.linear((x, x), torch.zeros(4, 16)),
                 lambda: layers.add_rms_norm(x, torch.ones(8)), lambda: layers.add_rms_norm_q8(x, torch.ones(8), x),
                 lambda: layers.linear_q8(x.to(torch.float8_e4m3fn), torch.ones(3), w.to(torch.float8_e4m3fn), torch.ones(4))):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="x must be"):
        layers.linear([1.0], w)
    with pytest.raises(TypeError, match="weight must be"):
        layers.linear(x, 3)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        layers.linear(x.double(), w.double())
    with pytest.raises(ValueError, match="at least one dimension"):
        layers.linear(torch.zeros(()), w)
    with pytest.raises(ValueError, match="residual has leading shape"):
        layers.linear(x, w, residual=torch.zeros(1, 4))
    with pytest.raises(ValueError, match="pieces of x"):
        layers.linear((x, x[:2]), w)
    with pytest.raises(ValueError, match="unknown activation"):
        hip.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="does not match x"):
        layers.add_rms_norm(x, torch.ones(8), x[:1])
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        layers.linear_q8(x, torch.ones(3), w.to(torch.float8_e4m3fn), torch.ones(4))
    with pytest.raises(ValueError, match="x_scale must be of shape"):
        layers.linear_q8(x.to(torch.float8_e4m3fn), torch.ones(3, 1), w.to(torch.float8_e4m3fn), torch.ones(4))
    with pytest.raises(NotImplementedError, match="no_grad"):
        layers.add_rms_norm_q8(x.requires_grad_(), torch.ones(8))


def test_python_entries_name_the_operand_that_is_no_tensor():
    x, w, f8 = torch.zeros(3, 8), torch.ones(8), torch.float8_e4m3fn
    for call, name in ((lambda: layers.add_rms_norm(3, w), "x"), (lambda: layers.add_rms_norm(x, 3), "weight"),
                       (lambda: layers.add_rms_norm(x, w, 3), "residual"), (lambda: layers.add_rms_norm_q8(x, w, [1]), "residual"),
                       (lambda: layers.linear(x, x, bias=3), "bias"), (lambda: layers.linear(x, x, residual=3), "residual"),
                       (lambda: layers.linear((x, 3), x), "the second piece of x"),
                       (lambda: layers.linear_q8(x.to(f8), 3, x.to(f8), torch.ones(3)), "x_scale"),
                       (lambda: layers.quantize_weight(3), "weight")):
        with pytest.raises(TypeError, match="%s must be a torch.Tensor" % name):
            call()
    for bad in (torch.zeros(8), torch.zeros(2, 3, 4), torch.zeros(4, 0)):
        with pytest.raises(ValueError, match="weight must be a matrix"):
            layers.quantize_weight(bad)


def test_quantize_weight_on_the_cpu():
    """Setup work in torch: runs anywhere.  Rows of zeros divide by the smallest scale."""
    w = torch.tensor([[0.0, 0.0], [448.0, 1.0], [-7.0, 3.5]])
    q, s = layers.quantize_weight(w)
    assert q.dtype == torch.float8_e4m3fn and s.tolist() == [2.0 ** -126, 1.0, 0.015625]
    assert torch.equal(q.float() * s[:, None], w)


def test_residual_networks_keep_the_reference_names_and_stay_off_the_fused_kernels():
    net = helpers.NeRF(D=8, W=256, input_ch=63, output_ch=4, skips=[4], input_ch_views=27, use_viewdirs=True)
    res = helpers.NeRF(D=8, W=256, input_ch=63, output_ch=4, skips=[4], input_ch_views=27, use_viewdirs=True, residual=True)
    assert net.hip_supported() and not res.hip_supported()
    assert [k for k in res.state_dict() if k not in net.state_dict()] == ["norm_weights.%d" % i for i in range(7)]
    assert list(net.state_dict()) == [k for k in res.state_dict() if not k.startswith("norm_weights")]
