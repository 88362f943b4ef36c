"""What the gated delta rule and group norm refuse, on the CPU: C entry points before any launch, and the Python surface."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_params_struct_matches_header(tmp_path):
    from openkimi_b200 import _lib

    fields = [f[0] for f in _lib.KdaGdrParams._fields_]
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "kda_b200.h"\nint main(){printf("%zu\\n", sizeof(KdaGdrParams));\n'
    prog += "".join(f'printf("%zu\\n", offsetof(KdaGdrParams, {f}));\n' for f in fields) + "return 0;}\n"
    src = tmp_path / "probe.c"
    src.write_text(prog)
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [C.sizeof(_lib.KdaGdrParams)] + [getattr(_lib.KdaGdrParams, f).offset for f in fields]


def _params():
    from openkimi_b200 import _lib

    p = _lib.KdaGdrParams()
    p.B, p.T, p.H, p.HV, p.dk, p.dv, p.N, p.NT, p.dtype, p.g_dtype = 1, 64, 1, 2, 128, 64, 1, 1, 1, 0
    for n in ("q", "k", "v", "g", "beta", "o", "workspace"):
        setattr(p, n, 4096)  # (never dereferenced)
    return p


@pytest.mark.parametrize("change,code", [(dict(dtype=7), 3), (dict(g_dtype=2), 3), (dict(dk=96), 2), (dict(dv=32), 2), (dict(HV=3, H=2), 2),
                                         (dict(NT=2), 2), (dict(N=2), 2), (dict(q=None), 1), (dict(o=None), 1), (dict(flags=2), 1),
                                         (dict(k=4100), 5), (dict(workspace=4112), 4), (dict(workspace_bytes=64), 4),
                                         (dict(cu_seqlens=4096), 1), (dict(T=0), 2)])
def test_entry_point_refusals(change, code):
    from openkimi_b200 import _lib

    lib = _lib.load()
    p = _params()
    fb, bb = C.c_size_t(), C.c_size_t()
    assert lib.kda_gdr_workspace_bytes(C.byref(p), C.byref(fb), C.byref(bb)) == 0 and fb.value and bb.value
    p.workspace_bytes = fb.value
    for n, v in change.items():
        setattr(p, n, v)
    assert lib.kda_gdr_fwd(C.byref(p), None) == code


def test_backward_refusals():
    from openkimi_b200 import _lib

    lib = _lib.load()
    p = _params()
    fb, bb = C.c_size_t(), C.c_size_t()
    assert lib.kda_gdr_workspace_bytes(C.byref(p), C.byref(fb), C.byref(bb)) == 0
    p.workspace_bytes = fb.value
    assert lib.kda_gdr_bwd(C.byref(p), None) == 1
    for n in ("grad_o", "grad_q", "grad_k", "grad_v", "grad_g", "grad_beta", "bwd_scratch"):
        setattr(p, n, 4096)
    assert lib.kda_gdr_bwd(C.byref(p), None) == 4                 # no scratch
    p.bwd_scratch_bytes = bb.value
    p.flags = _lib.FLAG_NO_SAVE
    assert lib.kda_gdr_bwd(C.byref(p), None) == 4                 # nothing was kept
    p.flags, p.A_log = _lib.FLAG_GATE, 4096
    assert lib.kda_gdr_bwd(C.byref(p), None) == 1                 # no place for dA_log
    p.flags, p.grad_q = 0, 4100
    assert lib.kda_gdr_bwd(C.byref(p), None) == 5
    assert lib.kda_gdr_fwd(None, None) == 1 and lib.kda_gdr_bwd(None, None) == 1


def test_recurrent_entry_refusals():
    from openkimi_b200 import _lib

    lib = _lib.load()

    def call(N=1, T=1, H=1, HV=2, dk=128, dv=64, dtype=1, g_dtype=1, flags=0, q=4096, state=4096, A=None):
        return lib.kda_gdr_recurrent_fwd(q, 4096, 4096, 4096, 4096, A, None, state, state, 4096, N, T, H, HV, dk, dv, dtype, g_dtype, flags, 1.0, None)

    assert call(q=None) == 1 and call(flags=2) == 1
    for bad in (dict(N=0), dict(T=0), dict(HV=3, H=2), dict(dk=32), dict(dv=256), dict(N=2 ** 30)):
        assert call(**bad) == 2, bad
    assert call(dtype=5) == 3 and call(g_dtype=5) == 3 and call(state=4104) == 5


def test_group_norm_entry_refusals():
    from openkimi_b200 import _lib

    lib = _lib.load()

    def fwd(x=4096, y=4096, mean=4096, N=2, S=3, ch=12, groups=4, eps=1e-5, dtype=1):
        return lib.kda_group_norm_fwd(x, None, None, y, mean, mean, mean, N, S, ch, groups, eps, 1, dtype, None)

    assert fwd(x=None) == 1 and fwd(y=None) == 1 and fwd(mean=None) == 1
    for bad in (dict(N=0), dict(S=0), dict(groups=5), dict(groups=0), dict(eps=-1.0), dict(eps=float("nan")), dict(N=2 ** 31)):
        assert fwd(**bad) == 2, bad
    assert fwd(dtype=3) == 3

    def bwd(dw=4096, db=4096, scratch=4096, dy=4096):
        return lib.kda_group_norm_bwd(4096, None, None, 4096, 4096, dy, 4096, dw, db, scratch, 2, 3, 12, 4, 1e-5, 1, 1, None)

    assert bwd(dy=None) == 1 and bwd(dw=None) == 1 and bwd(db=None) == 1 and bwd(scratch=None) == 1


def test_no_cpu_fallback():
    from openkimi_b200 import (chunk_gated_delta_rule, fused_recurrent_gated_delta_rule, group_norm, recurrent_gated_delta_rule_step)

    q, g = torch.zeros(1, 4, 1, 64), torch.zeros(1, 4, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        chunk_gated_delta_rule(q, q, q, g, g)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        chunk_gated_delta_rule(q, q, q, g, g, cu_seqlens=torch.tensor([0, 4]))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_recurrent_gated_delta_rule(q, q, q, g, g)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        recurrent_gated_delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], torch.zeros(1, 1, 64, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm(torch.zeros(4, 12), 3)
    with pytest.raises(ValueError, match="two offsets"):
        chunk_gated_delta_rule(q, q, q, g, g, cu_seqlens=torch.tensor([0]))
    with pytest.raises(ValueError, match="activation"):
        group_norm(torch.zeros(4, 12), 3, activation="tanh")


def test_module_refusals():
    from openkimi_b200 import FusedGroupNorm

    with pytest.raises(ValueError, match="divisible"):
        FusedGroupNorm(5, 12)
    with pytest.raises(ValueError, match="activation"):
        FusedGroupNorm(4, 12, activation="gelu")
    with pytest.raises(ValueError, match="last dimension"):
        FusedGroupNorm(4, 12)(torch.zeros(2, 13))
    m = FusedGroupNorm(4, 12, affine=False)
    assert m.weight is None and m.bias is None
