"""The C entry points of 16-bit cross attention that keep what the rounding of the result left off: refusals and workspaces, without
a GPU (every call ends at a check)."""
from q8_kernels_amd import _lib


def test_refusals_of_the_training_entry_points():
    L, B16 = _lib.lib(), _lib.Q8_BF16
    st = _lib._i64 * 3
    ok, odd = st(4096, 512, 64), st(4096, 512, 60)

    def fwd(q=16, qs=ok, o=16, low=16, lse=16, b=2, h=8, hk=8, m=8, n=8, d=64, dt=B16, ws=None, size=0):
        return L.q8_cross_attn_train(q, qs, 16, ok, 16, ok, o, ok, low, lse, None, None, 0, dt, 0.1, b, h, hk, m, n, d, ws, size, None)

    assert fwd(b=0, o=None, low=None, lse=None) == 0 and fwd(m=0, o=None, low=None, lse=None) == 0
    assert fwd(q=None) == -1 and fwd(o=None) == -1 and fwd(low=None) == -1 and fwd(lse=None) == -1 and fwd(n=100000) == -1
    assert fwd(low=24) == -4 and fwd(lse=18) == -4 and fwd(qs=odd) == -4 and fwd(d=60) == -3 and fwd(hk=3) == -3 and fwd(dt=_lib.Q8_F32) == -2
    assert fwd(b=1 << 20, h=16, hk=16, m=1) == -3

    def bwd(g=16, low=16, lse=16, dq=16, ws=16, size=1 << 40, b=2, h=8, m=8, n=300, d=64):
        return L.q8_cross_attn_train_backward(g, ok, 16, ok, 16, ok, 16, ok, 16, ok, low, lse, dq, ok, 16, ok, 16, ok, None, None, 0, B16, 0.1, b, h, h, m, n, d, ws, size,
                                              None)

    assert bwd(b=0, low=None) == 0 and bwd(m=0, n=0, low=None) == 0
    assert bwd(low=None) == -1 and bwd(g=None) == -1 and bwd(lse=None) == -1 and bwd(dq=None) == -1 and bwd(ws=None) == -1
    assert bwd(low=24) == -4 and bwd(ws=20) == -4 and bwd(size=16) == -3 and bwd(d=12) == -3 and bwd(b=1 << 20, h=16) == -3


def test_workspaces():
    """The backward that forms o_low itself takes that (a byte an element), and behind it the larger of what the forward and the
    other backward take."""
    L = _lib.lib()
    for b, h, hk, m, n, d in ((2, 8, 2, 70, 100, 64), (1, 32, 8, 1, 8192, 128), (3, 4, 4, 1000, 3000, 96), (1, 1, 1, 1, 1, 8), (2, 4, 4, 5, 0, 64), (2, 4, 4, 0, 5, 64)):
        with_low, without = (f(b, h, hk, m, n, d) for f in (L.q8_cross_attn_train_backward_workspace, L.q8_cross_attn_backward_workspace))
        assert with_low >= 0 and without == (b * h * m * d + 15) // 16 * 16 + max(with_low, L.q8_cross_attn_workspace(b, h, hk, m, n, d))
    assert L.q8_cross_attn_train_backward_workspace(2, 8, 3, 8, 8, 64) == -3
