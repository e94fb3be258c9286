"""Layer operators without a GPU: what the entry points refuse, before anything is launched, and the modules' initial values."""
import ctypes

import pytest
import torch
from torch import nn

from nrhints_amd import _lib, layers, ops


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) // 16 * 16            # never reached by a launch

    def fwd(dtype=0, x=p, ldx=8, w=p, ldw=8, b=None, r=None, ldr=0, act=0, beta=1.0, m=4, n=4, k=8, y=p, ldy=4, d=None):
        return lib.nrh_linear_forward(dtype, x, ldx, w, ldw, b, r, ldr, act, beta, m, n, k, y, ldy, d, None, 0, None)

    def data(dtype=0, g=p, ldg=4, d=None, ldd=0, act=0, w=p, ldw=8, m=4, n=4, k=8, o=p, ldo=8):
        return lib.nrh_linear_backward_data(dtype, g, ldg, d, ldd, act, w, ldw, m, n, k, o, ldo, None, 0, None)

    for bad in (dict(dtype=3), dict(dtype=-1), dict(act=6), dict(act=-1), dict(m=-1), dict(n=0), dict(k=0), dict(ldx=7), dict(ldw=7), dict(ldy=3),
                dict(x=None), dict(w=None), dict(y=None), dict(r=p, ldr=3), dict(act=2, beta=0.0), dict(act=2, beta=float("nan")), dict(x=p + 2),
                dict(dtype=1, w=p + 1), dict(b=p + 1), dict(m=1 << 31), dict(n=1 << 21), dict(k=1 << 21, ldx=1 << 21, ldw=1 << 21)):
        assert fwd(**bad) == -1, bad
        assert lib.nrh_last_error_string()
    assert fwd(m=0, x=None, y=None) == 0                   # no rows: nothing to do
    for bad in (dict(act=1), dict(d=p, ldd=4), dict(act=4, d=p, ldd=3), dict(ldo=7), dict(ldg=3), dict(g=None), dict(o=None), dict(m=1 << 31)):
        assert data(**bad) == -1, bad
    assert lib.nrh_linear_workspace_bytes(3, 0, 0, 1, 1, 1) == -1 and lib.nrh_linear_workspace_bytes(0, 0, 0, 1, 0, 1) == -1
    need = lib.nrh_linear_workspace_bytes(2, 0, 0, 100000, 256, 256)
    assert need > 0
    assert lib.nrh_linear_backward_weight(0, p, 256, None, 0, 0, p, 256, 100000, 256, 256, p, 256, None, None, 0, None) == -3
    assert lib.nrh_linear_backward_weight(0, p, 256, None, 0, 0, p, 256, 100000, 256, 256, p, 256, None, p, need - 1, None) == -3

    def emb(dtype=0, t=p, ldt=4, v=3, d=4, i=p, bits=64, n=2, o=p, ldo=4):
        return lib.nrh_embedding_forward(dtype, t, ldt, v, d, i, bits, n, 1.0, o, ldo, None)

    for bad in (dict(dtype=5), dict(t=None), dict(ldt=3), dict(v=0), dict(d=0), dict(i=None), dict(bits=16), dict(n=-1), dict(ldo=3), dict(o=None),
                dict(i=p + 4), dict(n=(1 << 30) + 1), dict(v=1 << 31), dict(t=p + 2)):
        assert emb(**bad) == -1, bad
    assert emb(n=0, i=None, o=None) == 0
    assert lib.nrh_embedding_backward(0, p, 4, p, 64, 2, 300, 4, 1.0, p, 4, None, 0, None) == -3
    assert lib.nrh_embedding_backward(0, p, 4, p, 64, 2, 3, 4, 1.0, None, 4, None, 0, None) == -1
    assert lib.nrh_embedding_backward_workspace_bytes(-1, 3, 4) == -1 and lib.nrh_embedding_backward_workspace_bytes(0, 3, 4) == 0


def test_workspace_sizes_cover_every_shape():
    """The workspace is a multiple of the partial outputs it holds and never negative, over a sweep of sizes."""
    lib = _lib.load()
    for m in (0, 1, 17, 300, 4096, 163840, 655360, 1 << 30):
        for n in (1, 3, 64, 129, 256, 1024):
            for k in (1, 39, 84, 256, 361, 4096):
                for dtype, act in ((0, 0), (1, 0), (2, 0), (2, 1), (1, 4)):
                    for op, out in ((0, m * n), (1, m * k), (2, n * k + n)):
                        b = lib.nrh_linear_workspace_bytes(op, dtype, act, m, n, k)
                        assert b >= 0 and (b == 0 or (b % (4 * out) == 0 and b // (4 * out) <= 512 and b < 1 << 31)), (op, m, n, k, b)


def test_no_cpu_path():
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    for call in (lambda: ops.linear(x, w), lambda: ops.embedding(w, torch.zeros(2, dtype=torch.int64)), lambda: layers.linear(x, w),
                 lambda: layers.Linear(4, 5)(x), lambda: layers.Embedding(3, 4)(torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.embedding_backward(x, torch.zeros(3, dtype=torch.int64), 5)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_modules_initialise_like_torch():
    torch.manual_seed(3)
    a, e = layers.Linear(7, 5, activation="relu"), layers.Embedding(6, 4)
    torch.manual_seed(3)
    b, f = nn.Linear(7, 5), nn.Embedding(6, 4)
    assert torch.equal(a.weight, b.weight) and torch.equal(a.bias, b.bias) and torch.equal(e.weight, f.weight)
    assert layers.Linear(7, 5, bias=False).bias is None and set(a.state_dict()) == {"weight", "bias"}
    for bad in (lambda: layers.Linear(0, 3), lambda: layers.Linear(3, 3, activation="tanh"), lambda: layers.Embedding(0, 3)):
        with pytest.raises(ValueError):
            bad()


def test_background_network_shapes():
    """outside_nerf beyond the compiled shape is accepted (layers.linear), with the reference's layer sizes; what no layer chain can run
    and networks narrower than the compiled one are refused."""
    import nrhints_amd as na
    on = na.NeuSRendererConfig(use_outside_nerf=True)
    wide = na.NeuSModelConfig(renderer=on, outside_nerf=na.NeRFConfig(d_hidden=512, n_layers=6, multi_res=8, multi_res_view=3, skips=[2, 4]))
    assert na.unsupported_reason(wide) is None
    m = na.NeuSHintRenderer(wide).outside_nerf
    assert not m.compiled and na.NeuSHintRenderer(na.NeuSModelConfig(renderer=on)).outside_nerf.compiled
    ch, cv = 4 * 17, 6 * 7
    assert [tuple(l.weight.shape) for l in m.pts_linears] == [(512, ch), (512, 512), (512, 512), (512, 512 + ch), (512, 512), (512, 512 + ch)]
    assert m.views_linears[0].weight.shape == (256, 512 + cv) and m.alpha_linear.weight.shape == (1, 512) and m.rgb_linear.weight.shape == (3, 256)
    with pytest.raises(RuntimeError, match="GPU only"):
        m(torch.zeros(4, 4), torch.zeros(1, 3), torch.zeros(1, 3), pts_per_ray=4)
    for bad in (dict(d_hidden=300, n_layers=4, skips=[3]), dict(d_hidden=257), dict(d_hidden=255), dict(d_hidden=64), dict(skips=[7]), dict(skips=[-1]), dict(multi_res=0),
                dict(n_layers=1, skips=[])):
        assert na.unsupported_reason(na.NeuSModelConfig(renderer=on, outside_nerf=na.NeRFConfig(**bad))), bad
        # (off by default: a network that is not built is not looked at)
        assert na.unsupported_reason(na.NeuSModelConfig(outside_nerf=na.NeRFConfig(**bad))) is None
