"""CPU checks of the joiner's operators: what is refused, and with which error.  No kernel is launched."""
import pytest
import torch

import warp_ctct_b200 as W


@pytest.fixture(scope="module")
def lib():
    from warp_ctct_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="must be located in the CUDA"):
        W.layer_norm(x)
    with pytest.raises(RuntimeError, match="must be located in the CUDA"):
        W.joint_layer_norm(x.view(1, 4, 8), x.view(1, 4, 8))
    with pytest.raises(RuntimeError, match="must be located in the CUDA"):
        W.adjust_logits(x)
    with pytest.raises(RuntimeError, match="must be located in the CUDA"):
        W.adjust_joint_logits(torch.randn(1, 2, 3, 4), torch.ones(1, 2, dtype=torch.int32))


def test_pack_token_mask_words():
    mask = torch.zeros(2, 70, dtype=torch.bool)
    mask[0, 0] = mask[0, 31] = mask[0, 33] = mask[1, 69] = True
    words = W.pack_token_mask(mask)
    assert words.dtype == torch.int32 and words.shape == (2, 3)
    assert words.tolist() == [[1 - 2 ** 31, 2, 0], [0, 0, 1 << 5]]
    g = torch.Generator().manual_seed(0)
    mask = torch.rand(3, 5, 129, generator=g) < 0.5
    words = W.pack_token_mask(mask)
    v = torch.arange(129)
    assert torch.equal(((words[..., v // 32] >> (v % 32)) & 1).bool(), mask)


def test_layer_norm_entry_points_refuse_bad_arguments(lib):
    p = 4096  # an address that is never dereferenced: every call below is refused before a launch
    assert lib.ctct_b200_layer_norm_workspace_bytes(-1, 8, 0) == 0
    assert lib.ctct_b200_layer_norm_workspace_bytes(4, 0, 0) == 0
    assert lib.ctct_b200_layer_norm_workspace_bytes(4, 8, 3) == 0
    assert lib.ctct_b200_layer_norm_workspace_bytes(1, 8, 0) >= 64
    fwd, bwd = lib.ctct_b200_layer_norm_forward, lib.ctct_b200_layer_norm_backward
    assert fwd(None, 8, 0, 4, 8, None, None, 1, 1e-5, p, None, None) == -1
    assert fwd(p, 8, 0, 4, 8, None, None, 1, 1e-5, None, None, None) == -1
    assert fwd(p, 8, 5, 4, 8, None, None, 1, 1e-5, p, None, None) == -1
    assert fwd(p, 8, 0, 4, 0, None, None, 1, 1e-5, p, None, None) == -1
    assert fwd(p, 8, 0, -1, 8, None, None, 1, 1e-5, p, None, None) == -1
    assert fwd(None, 8, 0, 0, 8, None, None, 1, 1e-5, None, None, None) == 0   # no row: nothing to do
    assert bwd(p, 8, p, 8, 0, 4, 8, p, 1, None, p, p, p, p, 1 << 20, None) == -1
    assert bwd(p, 8, p, 8, 0, 4, 8, p, 1, p, p, p, p, None, 0, None) == -2
    assert bwd(p, 8, p, 8, 0, 4, 8, p, 1, p, p, p, p, p + 8, 1 << 20, None) == -2  # misaligned
    assert bwd(p, 8, p, 8, 0, 4, 8, p, 1, p, p, p, p, p, 8, None) == -2            # too small


def test_joint_norm_entry_points_refuse_bad_arguments(lib):
    p = 4096
    assert lib.ctct_b200_joint_norm_saved_bytes(2, 3, 0, -1, 1) == 0
    assert lib.ctct_b200_joint_norm_saved_bytes(2, 3, 4, -1, 0) == 0   # nothing is kept without a gradient
    assert lib.ctct_b200_joint_norm_saved_bytes(2, 3, 4, 10, 0) >= 24
    assert lib.ctct_b200_joint_norm_saved_bytes(2, 3, 4, -1, 1) >= 4 * (6 + 8 + 24)
    assert lib.ctct_b200_joint_norm_workspace_bytes(2, 3, 4, 8193, 0) == 0
    assert lib.ctct_b200_joint_norm_workspace_bytes(2, 3, 4, 8192, 0) > 0

    def fwd(f=p, g=p, dtype=0, lx=p, ly=p, N=2, T=3, U1=4, H=8, rows=-1, y=p, grad=0, saved=None, nbytes=0):
        return lib.ctct_b200_joint_norm_forward(f, T * H, H, g, U1 * H, H, dtype, lx, ly, N, T, U1, H, rows, None, None, 1, 1e-5, y,
                                                grad, saved, nbytes, None)

    assert fwd(f=None) == -1 and fwd(g=None) == -1 and fwd(y=None) == -1 and fwd(dtype=7) == -1
    assert fwd(N=70000) == -1 and fwd(U1=0) == -1 and fwd(H=0) == -1 and fwd(T=-1) == -1
    assert fwd(rows=5, lx=None) == -1
    assert fwd(rows=5) == -2 and fwd(grad=1) == -2 and fwd(grad=1, saved=p, nbytes=8) == -2
    assert fwd(grad=1, saved=p + 4, nbytes=1 << 20) == -2
    assert fwd(H=8193) == -4
    assert fwd(N=0) == 0 and fwd(T=0) == 0 and fwd(rows=0) == 0
    bwd = lib.ctct_b200_joint_norm_backward
    ok = [p, p, 24, 8, p, 32, 8, 0, p, p, 2, 3, 4, 8, -1, p, 1, p, 1 << 20, p, p, p, p, p, 1 << 24, None]
    for i, bad, rc in ((0, None, -1), (1, None, -1), (7, 9, -1), (17, None, -2), (18, 4, -2), (23, None, -2), (24, 4, -2),
                       (23, p + 8, -2), (13, 20000, -4)):
        args = list(ok)
        args[i] = bad
        assert bwd(*args) == rc, (i, bad)


def test_adjust_entry_points_refuse_bad_arguments(lib):
    p = 4096
    assert lib.ctct_b200_adjust_workspace_bytes(2, 3, 4, 5, 0, 0, 2) >= 2 * 4 * 5 * 4
    assert lib.ctct_b200_adjust_workspace_bytes(2, 3, 1 << 16, 1 << 16, 0, 0, 2) == 0   # a plane beyond 2^31 elements

    def fwd(x=p, stride=0, dtype=0, tok=p, pitch=3, lens=None, lx=None, ly=None, N=2, T=3, U1=4, V=8, rows=-1, cu=None, bias=None,
            bk=0, allowed=None, mk=0, rho=1.0, rho_n=None, out=p):
        return lib.ctct_b200_adjust_forward(x, stride, dtype, tok, pitch, lens, lx, ly, N, T, U1, V, rows, cu, bias, bk, 1, allowed,
                                            mk, rho, 0.0, 0.0, rho_n, None, None, out, None)

    assert fwd(x=None) == -1 and fwd(out=None) == -1 and fwd(dtype=4) == -1 and fwd(V=0) == -1 and fwd(N=-1) == -1
    assert fwd(rho=0.0) == -1 and fwd(rho=float("nan")) == -1
    assert fwd(bk=1) == -1 and fwd(bias=p) == -1 and fwd(mk=1) == -1 and fwd(allowed=p) == -1 and fwd(bias=p, bk=4) == -1
    assert fwd(pitch=2) == -1            # labels shorter than the contexts
    assert fwd(stride=8) == -1           # a row stride belongs to a step
    assert fwd(rows=5, cu=p) == -1 and fwd(rows=5, lx=p, ly=p) == -1
    assert fwd(N=0) == 0 and fwd(T=0) == 0 and fwd(rows=0, lx=p, ly=p, cu=p) == 0
    ok = [p, p, 0, 0, p, 3, None, None, None, 2, 3, 4, 8, -1, None, 1, 1, None, 0, 1.3, None, p, p, p, 1 << 20, None]
    for i, bad, rc in ((0, None, -1), (1, None, -1), (3, 4, -1), (15, 0, -1), (15, 9, -1), (23, None, -2), (24, 4, -2), (23, p + 8, -2)):
        args = list(ok)
        args[i] = bad
        assert lib.ctct_b200_adjust_backward(*args) == rc, (i, bad)


def test_frames_near_the_end_of_32_bits_are_refused(lib):
    """Frame counters step past the last frame by up to a block's share: that must not wrap."""
    p = 4096
    for T in (2 ** 31 - 1, 2 ** 31 - 4096):
        assert lib.ctct_b200_adjust_forward(p, 0, 0, None, 0, None, None, None, 1, T, 1, 1, -1, None, None, 0, 1, None, 0, 1.0, 0.0, 0.0,
                                            None, None, None, p, None) == -1
        assert lib.ctct_b200_adjust_workspace_bytes(1, T, 1, 1, 0, 0, 1) == 0
        assert lib.ctct_b200_joint_norm_forward(p, T, 1, p, 1, 1, 0, None, None, 1, T, 1, 1, -1, None, None, 1, 1e-5, p, 0, None, 0,
                                                None) == -1
        assert lib.ctct_b200_joint_norm_workspace_bytes(1, T, 1, 1, 0) == 0


def test_gradients_that_are_not_aligned_are_refused(lib):
    """Sums are stored as vectors."""
    p = 4096
    ok = [p, p, 24, 8, p, 32, 8, 0, p, p, 2, 3, 4, 8, -1, p, 1, p, 1 << 20, p, p, p, p, p, 1 << 24, None]
    for i in (19, 20):
        args = list(ok)
        args[i] = p + 4
        assert lib.ctct_b200_joint_norm_backward(*args) == -1
    ok = [p, p, 0, 0, p, 3, None, None, None, 2, 3, 4, 8, -1, None, 1, 1, None, 0, 1.3, None, p, p, p, 1 << 20, None]
    args = list(ok)
    args[22] = p + 4
    assert lib.ctct_b200_adjust_backward(*args) == -1
