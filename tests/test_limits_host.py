"""Sizes past what a launch takes are refused by the C entries before any launch."""
from esr_amd import _lib

E = -1  # ESR_EINVAL
P = 1 << 20  # never dereferenced


def test_group_norm_channels():
    lib = _lib.load()
    for C, off in ((1 << 24, 4), ((1 << 24) - 1, 0), (65535 * 256 + 1, 0)):  # 65536 chunks of 256 channels
        x = P + off
        for HW in (1, 1 << 13):
            ok = (1, HW, C, 1)
            assert lib.esr_gn_workspace_bytes(*ok) > 0
            assert lib.esr_gn_lrelu_fwd(x, *ok, None, None, 1e-5, 0.2, P, P, None, None, None, None, P, None) == E
            assert lib.esr_gn_lrelu_bwd(x, None, None, P, *ok, None, None, P, 0.2, P, P, P, P, P, None) == E
            assert lib.esr_gn_lrelu_bwd2(x, None, None, P, None, None, None, *ok, None, None, P, 0.2, P, P, P, P, P,
                                         None) == E
