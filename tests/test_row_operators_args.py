"""Refusals of the row operators (rms_norm, log_probs, adamw_update) and their workspace sizes: argument checks come
before anything touches a device, so they run without one.  The addresses here are never dereferenced."""
import ctypes as C

import pytest
import torch

from pixienn_b200 import capi, ops

A, B_, C_, D, E, F = (0x10000000 * k for k in range(1, 7))


def refused(rc, word, status=capi.PXE_ERR_BAD_ARG):
    msg = capi.lib().pxe_last_error_string().decode()
    assert rc == status and word in msg, (rc, msg)


def norm(**kw):
    d = capi.RmsNormDesc()
    d.x, d.y, d.rstd, d.rows, d.channels, d.type, d.eps = A, B_, C_, 8, 64, capi.BF16, 1e-6
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.lib().pxe_rms_norm(None, C.byref(d))


def test_rms_norm_refusals():
    L = capi.lib()
    refused(L.pxe_rms_norm(None, None), "null descriptor")
    refused(norm(type=7), "unknown type")
    refused(norm(weight=D, weight_type=capi.F16), "weight_type")
    refused(norm(rows=-1), "shape")
    refused(norm(channels=0), "shape")
    refused(norm(channels=300000), "at most", capi.PXE_ERR_UNSUPPORTED)
    refused(norm(y=None), "exactly one")
    refused(norm(q=D, scale=E), "exactly one")
    refused(norm(y=None, q=D), "without scale")
    refused(norm(y=None, q=D, scale=E, group=48), "group")
    refused(norm(eps=-1.0), "eps")
    refused(norm(eps=float("nan")), "eps")
    refused(norm(x=None), "x is null")
    refused(norm(residual=D), "come together")
    refused(norm(h=D), "come together")
    refused(norm(x_row_stride=63), "x_row_stride")
    refused(norm(x=A + 1), "not aligned")
    refused(norm(weight=D + 2, weight_type=capi.F32), "not aligned")
    refused(norm(y=A + 64), "partially overlaps")
    refused(norm(y=A, y_row_stride=128), "partially overlaps")              # the same memory with another stride
    refused(norm(residual=D, h=D + 2), "partially overlaps")
    refused(norm(residual=D, h=B_), "y overlaps h")
    refused(norm(y=None, q=A, scale=E), "q overlaps x")
    refused(norm(rstd=A + 32), "rstd or scale overlaps")
    refused(norm(y=None, q=D, scale=A), "rstd or scale overlaps")
    refused(norm(y=None, q=D, scale=C_ + 4), "rstd, scale and weight overlap")
    refused(norm(weight=B_, weight_type=capi.F32), "y overlaps the weight")
    refused(norm(rstd=C_ + 2), "not aligned")
    assert norm(rows=0) == capi.PXE_OK and norm(rows=0, x=None, rstd=None) == capi.PXE_OK


def back(**kw):
    d = capi.RmsNormBackwardDesc()
    d.dy, d.h, d.rstd, d.dx, d.rows, d.channels, d.type = A, B_, C_, D, 8, 64, capi.F16
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.lib().pxe_rms_norm_backward(None, C.byref(d))


def test_rms_norm_backward_refusals_and_workspace():
    L = capi.lib()
    refused(L.pxe_rms_norm_backward(None, None), "null descriptor")
    refused(back(dy=None), "null pointer")
    refused(back(rstd=None), "null pointer")
    refused(back(dx=A + 128), "partially overlaps dy")
    refused(back(dresidual=E, dx=E + 2), "partially overlaps dresidual")
    refused(back(dweight=E), "workspace")
    refused(back(dweight=E, workspace=F + 4, workspace_bytes=1 << 20), "aligned workspace")
    refused(back(dweight=E, workspace=F, workspace_bytes=64), "needed", capi.PXE_ERR_WORKSPACE)
    refused(back(dweight=E + 2, workspace=F, workspace_bytes=1 << 20), "not aligned")
    refused(back(dweight=A + 4, workspace=F, workspace_bytes=1 << 20), "overlaps dy")
    refused(back(dweight=F + 64, workspace=F, workspace_bytes=1 << 20), "overlaps dweight")
    refused(back(channels=1 << 20), "at most", capi.PXE_ERR_UNSUPPORTED)
    refused(back(dx=C_), "overlaps rstd")
    refused(back(dweight=C_, workspace=F, workspace_bytes=1 << 20), "overlaps rstd")
    refused(back(weight=E, weight_type=capi.F32, dweight=E, workspace=F, workspace_bytes=1 << 20), "overlaps rstd or the weight")
    assert back(rows=0, dy=None) == capi.PXE_OK
    need = L.pxe_rms_norm_backward_workspace_bytes
    assert need(0, 64) == 0 and need(3, 64) == 3 * 64 * 4 and need(1 << 30, 1023) == 1184 * 1023 * 4 and need(1 << 30, 16384) == 148 * 16384 * 4


def probs(**kw):
    d = capi.LogProbsDesc()
    d.x, d.target, d.logp, d.entropy, d.stats = A, B_, C_, D, E
    d.rows, d.classes, d.type, d.temperature = 8, 100, capi.F32, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.lib().pxe_log_probs(None, C.byref(d))


def test_log_probs_refusals():
    L = capi.lib()
    refused(L.pxe_log_probs(None, None), "null descriptor")
    refused(probs(type=-1), "unknown type")
    refused(probs(classes=0), "shape")
    refused(probs(classes=0x7fffffff), "too many classes")
    refused(probs(rows=1 << 31), "too many rows")
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-31, 1e31):
        refused(probs(temperature=t), "temperature")
    refused(probs(top=33, top_logp=F, top_index=F + 4096), "top 33")
    refused(probs(top=5, classes=4, top_logp=F, top_index=F + 4096), "top 5")
    refused(probs(top=-1), "top -1")
    refused(probs(top=5), "come with top")
    refused(probs(top_logp=F), "come with top")
    refused(probs(x=None), "x is null")
    refused(probs(target=None), "come together")
    refused(probs(logp=None), "come together")
    refused(probs(x=A + 2), "not aligned")
    refused(probs(row_stride=99), "row stride")
    refused(probs(inner=3), "groups of 3")
    refused(probs(inner=4, outer_stride=300), "outer stride")
    refused(probs(entropy=A + 400), "overlaps")
    refused(probs(entropy=B_), "overlaps")
    refused(probs(entropy=B_ + 28), "overlaps an input")
    refused(probs(entropy=C_ + 4), "two outputs overlap")
    refused(probs(entropy=D + 2), "not aligned")
    assert probs(rows=0, x=None) == capi.PXE_OK


def probs_back(**kw):
    d = capi.LogProbsBackwardDesc()
    d.x, d.target, d.stats, d.dlogp, d.dx = A, B_, C_, D, E
    d.rows, d.classes, d.type, d.temperature = 8, 100, capi.F32, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.lib().pxe_log_probs_backward(None, C.byref(d))


def test_log_probs_backward_refusals():
    L = capi.lib()
    refused(L.pxe_log_probs_backward(None, None), "null descriptor")
    refused(probs_back(stats=None), "null pointer")
    refused(probs_back(dlogp=None), "neither")
    refused(probs_back(target=None), "neither")
    refused(probs_back(target=None, dentropy=F), "dlogp without target")
    refused(probs_back(dx=A + 4), "partially overlaps x")
    refused(probs_back(dx=A, dx_row_stride=200), "partially overlaps x")
    refused(probs_back(dx=C_), "overlaps an input")
    refused(probs_back(dx=A + 4 * 150, row_stride=200, dx_row_stride=200), "partially overlaps x")        # columns 150..250 of rows of 200
    refused(probs_back(dx=A + 4 * 950, inner=4, outer_stride=1500, dx_outer_stride=1500, row_stride=300, dx_row_stride=300), "partially overlaps x")
    refused(probs_back(dx_row_stride=50), "row stride")
    refused(probs_back(temperature=0.0), "temperature")
    assert probs_back(rows=0, x=None) == capi.PXE_OK


def adamw(entries, **kw):
    arr = (capi.AdamwTensor * max(1, len(entries)))()
    for row, t in zip(arr, entries):
        row.param, row.grad, row.m, row.v, row.n = A, B_, C_, D, 1000
        for k, v in t.items():
            setattr(row, k, v)
    d = capi.AdamwDesc()
    d.tensors, d.count, d.state_bits, d.t = C.addressof(arr), len(entries), 32, 1
    d.rate, d.beta1, d.beta2, d.eps, d.grad_scale = 1e-3, 0.9, 0.999, 1e-8, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.lib().pxe_adamw_update(None, C.byref(d))


def test_adamw_refusals():
    L = capi.lib()
    refused(L.pxe_adamw_update(None, None), "null descriptor")
    refused(adamw([{}], count=-1), "list of tensors")
    refused(adamw([{}], tensors=None), "list of tensors")
    refused(adamw([{}], param_type=9), "unknown type")
    refused(adamw([{}], param_type=capi.BF16, grad_type=capi.F16), "16-bit", capi.PXE_ERR_UNSUPPORTED)
    refused(adamw([{}], state_bits=16), "state_bits")
    refused(adamw([{}], beta1=1.0), "beta1")
    refused(adamw([{}], beta2=float("nan")), "beta1")
    refused(adamw([{}], eps=-1e-8), "eps")
    refused(adamw([{}], t=0), "step 0")
    refused(adamw([{"n": -1}]), "-1 elements")
    refused(adamw([{"grad": None}]), "null pointer")
    refused(adamw([{}], state_bits=8), "scales come with")
    refused(adamw([{"m_scale": E, "v_scale": F}]), "scales come with")
    refused(adamw([{"master": E}]), "master copy of fp32")
    refused(adamw([{"master": E}, {"param": F}], param_type=capi.BF16), "in all tensors or in none")
    refused(adamw([{"param": A + 2}]), "not aligned")
    refused(adamw([{}, {"grad": E, "m": F, "v": F + 8000}]), "overlap")                     # one parameter twice
    refused(adamw([{"m": A + 4}]), "overlap")
    refused(adamw([{"grad": A}]), "overlap")
    refused(adamw([{"v": C_}]), "overlap")
    refused(adamw([{}, {"param": E, "grad": B_ + 8000, "m": C_ + 3996, "v": F}]), "overlap")
    assert adamw([]) == capi.PXE_OK
    assert adamw([{"n": 0, "param": None, "grad": None}]) == capi.PXE_OK


def test_struct_layouts_match_the_header(tmp_path):
    """sizeof of every descriptor, as gcc lays it out."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"pxe_rms_norm_desc": capi.RmsNormDesc, "pxe_rms_norm_backward_desc": capi.RmsNormBackwardDesc,
             "pxe_log_probs_desc": capi.LogProbsDesc, "pxe_log_probs_backward_desc": capi.LogProbsBackwardDesc,
             "pxe_adamw_tensor": capi.AdamwTensor, "pxe_adamw_desc": capi.AdamwDesc}
    lines = []
    for n, cls in names.items():
        lines.append(f'printf("%zu\\n", sizeof({n}));')
        lines += [f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "sizes.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"pxe.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in names.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_operators_refuse_cpu_tensors_and_bad_rows():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm_e4m3(x), lambda: ops.rms_norm_backward(x, x, None, x[:, 0]),
                 lambda: ops.log_probs(x), lambda: ops.log_probs_backward(x, None, x), lambda: ops.AdamW([x])):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        ops.rms_norm_e4m3(x, group=16)
    stride = lambda t: ops._row_stride(t, "x")  # noqa: E731
    assert stride(torch.zeros(3, 5, 7)) == 7 and stride(torch.zeros(3, 5, 9)[..., :7]) == 9 and stride(torch.zeros(7)) == 7
    assert stride(torch.zeros(2, 6, 4, 4).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)) == 6
    for bad in (torch.zeros(5, 7).t(), torch.zeros(3, 6, 7)[:, :5], torch.zeros(1, 7).expand(4, 7), torch.zeros(4).as_strided((2, 3), (1, 1))):
        with pytest.raises(ValueError):
            stride(bad)
    assert ops._grouped_rows(torch.zeros(3, 6, 7)[:, :5], "x") == (5, 42, 7)
    assert ops._grouped_rows(torch.zeros(3, 6, 7), "x") == (6, 42, 7)
    assert ops._grouped_rows(torch.zeros(1, 6, 7)[:, 1:], "x") == (0, 0, 7)
    empty = ops.AdamW([])
    empty.step([], rate=1e-3, t=1)
    with pytest.raises(ValueError):
        empty.step([x], rate=1e-3, t=1)
