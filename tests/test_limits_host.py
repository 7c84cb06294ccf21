"""Sizes past what a launch takes are refused by the C entries before any launch."""
import os
import subprocess

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


def test_weight_gradient_grids():
    """64·65536 rows of the reduction, or a workgroup per 64 x 64 weights and tap, beyond 2^32 threads."""
    lib = _lib.load()
    for geo in ((1, 8, 8, 65536, 1, 1, 65536, 8, 1, 0), (1, 7, 7, 65536, 1, 1, 65536, 7, 1, 0)):
        assert lib.esr_dconv_wgrad_act8_workspace_bytes(*geo) == E
        assert lib.esr_dconv_wgrad_act8(P, P, *geo[:4], P, *geo[4:], P, P, None) == E
    assert lib.esr_dconv_wgrad_act8_workspace_bytes(1, 8, 8, 4096, 1, 1, 4096, 8, 1, 0) > 0


def test_weight_gradient_workgroups(tmp_path):
    """The workgroups of a grid of splits x items take every (split, item) once, whatever their numbers: none is idle, so
    that the 8 XCDs (ids modulo 8) differ by one workgroup at most.  Of every eight splits, one is one XCD's."""
    src = tmp_path / 'place.cpp'
    src.write_text('#include "esr_wgrad8_map.h"\n#include <cstdio>\n#include <initializer_list>\nint main() {\n'
                   '    for (int s = 1; s < 70; ++s)\n        for (int w : {1, 2, 3, 8, 16, 100, 128})\n'
                   '            for (int i = 0; i < s * w; ++i) {\n'
                   '                const auto p = wgrad8::place(i, s, w);\n'
                   '                std::printf("%d %d %d %d %d\\n", s, w, i, p.split, p.item);\n            }\n}\n')
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), '..', 'csrc')
    subprocess.run(['g++', '-std=c++17', '-I', csrc, str(src), '-o', str(tmp_path / 'place')], check=True)
    out = subprocess.run([str(tmp_path / 'place')], capture_output=True, text=True, check=True).stdout
    seen = {}
    for line in out.splitlines():
        s, w, i, split, item = map(int, line.split())
        assert 0 <= split < s and 0 <= item < w
        seen.setdefault((s, w), {})[split, item] = i
    for (s, w), at in seen.items():
        assert len(at) == s * w
        for split in range(s // 8 * 8):
            assert len({at[split, item] % 8 for item in range(w)}) == 1
