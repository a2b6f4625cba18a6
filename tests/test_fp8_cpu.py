"""CPU: the 8-bit linear layer's entry points reject bad arguments before touching a device, their structures match the
header, and the oracle's 8-bit form agrees with torch's e4m3."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import vibekernel_b200 as vk
from oracle import fp8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUPPORTED, ALIGNMENT = vk.VK_ERR_INVALID_ARGUMENT, vk.VK_ERR_UNSUPPORTED, vk.VK_ERR_ALIGNMENT
P = 0x1000


def _call(name, **fields):
    args = {"quantize_fp8": vk.QuantizeFp8Args, "rmsnorm_fp8": vk.RmsnormFp8Args, "gemm_fp8": vk.GemmFp8Args,
            "rmsnorm_fp8_backward": vk.RmsnormFp8BackwardArgs, "wgrad_fp8": vk.WgradFp8Args}[name]()
    for k, v in fields.items():
        setattr(args, k, v)
    return getattr(vk.lib, "vk_" + name)(ctypes.byref(args))


def _good(name):
    return dict({
        "quantize_fp8": dict(X=P, Q=P, scale=P, rows=4, cols=8),
        "rmsnorm_fp8": dict(X=P, weight=P, Q=P, scale=P, rstd=P, rows=4, cols=8, eps=1e-6),
        "rmsnorm_fp8_backward": dict(dY=P, H=P, weight=P, rstd=P, dX=P, dweight=P, workspace=P, workspace_bytes=1 << 20,
                                     rows=4, cols=8),
        "gemm_fp8": dict(A=P, B=P, a_scale=P, b_scale=P, C=P, m=4, n=8, k=8, trans_b=1),
        "wgrad_fp8": dict(dY=P, X=P, x_scale=P, dW=P, tokens=4, n=8, k=8),
    }[name])


NAMES = ("quantize_fp8", "rmsnorm_fp8", "rmsnorm_fp8_backward", "gemm_fp8", "wgrad_fp8")


@pytest.mark.parametrize("name", NAMES)
def test_null_arguments(name):
    assert getattr(vk.lib, "vk_" + name)(None) == BAD
    assert "args is NULL" in vk.last_error()


@pytest.mark.parametrize("name,fields,code", [
    ("quantize_fp8", dict(rows=-1), BAD), ("quantize_fp8", dict(cols=-1), BAD), ("quantize_fp8", dict(dtype=3), BAD),
    ("quantize_fp8", dict(scaling=2), BAD), ("quantize_fp8", dict(ldx=7), BAD), ("quantize_fp8", dict(ldq=7), BAD),
    ("quantize_fp8", dict(ldx=-8), BAD), ("quantize_fp8", dict(ld_scale=1, cols=129, ldx=0), BAD),
    ("quantize_fp8", dict(rows=1 << 40), UNSUPPORTED), ("quantize_fp8", dict(ldx=1 << 50), UNSUPPORTED),
    ("quantize_fp8", dict(X=None), BAD), ("quantize_fp8", dict(Q=None), BAD), ("quantize_fp8", dict(scale=None), BAD),
    ("rmsnorm_fp8", dict(cols=0), BAD), ("rmsnorm_fp8", dict(rows=-1), BAD), ("rmsnorm_fp8", dict(dtype=1), BAD),
    ("rmsnorm_fp8", dict(eps=-1.0), BAD), ("rmsnorm_fp8", dict(eps=float("nan")), BAD),
    ("rmsnorm_fp8", dict(residual=P), BAD), ("rmsnorm_fp8", dict(H=P), BAD), ("rmsnorm_fp8", dict(rstd=None), BAD),
    ("rmsnorm_fp8", dict(weight=None), BAD), ("rmsnorm_fp8", dict(residual=P, H=P, ldh=7), BAD),
    ("rmsnorm_fp8_backward", dict(cols=0), BAD), ("rmsnorm_fp8_backward", dict(dtype=1), BAD),
    ("rmsnorm_fp8_backward", dict(workspace=None), BAD), ("rmsnorm_fp8_backward", dict(workspace_bytes=127), BAD),
    ("rmsnorm_fp8_backward", dict(workspace=P + 4), BAD), ("rmsnorm_fp8_backward", dict(dweight=None), BAD),
    ("rmsnorm_fp8_backward", dict(dX=None), BAD), ("rmsnorm_fp8_backward", dict(lddx=7), BAD),
    ("gemm_fp8", dict(m=-1), BAD), ("gemm_fp8", dict(k=1 << 31), UNSUPPORTED), ("gemm_fp8", dict(dtype=5), BAD),
    ("gemm_fp8", dict(trans_b=2), BAD), ("gemm_fp8", dict(a_scaling=2), BAD), ("gemm_fp8", dict(b_scaling=-1), BAD),
    ("gemm_fp8", dict(trans_b=0), UNSUPPORTED), ("gemm_fp8", dict(lda=7), BAD), ("gemm_fp8", dict(ldb=7), BAD),
    ("gemm_fp8", dict(ldc=7), BAD), ("gemm_fp8", dict(C=None), BAD), ("gemm_fp8", dict(a_scale=None), BAD),
    ("gemm_fp8", dict(k=300, ld_a_scale=2), BAD), ("gemm_fp8", dict(k=300, ld_b_scale=2), BAD),
    ("wgrad_fp8", dict(tokens=-1), BAD), ("wgrad_fp8", dict(dtype=1), BAD), ("wgrad_fp8", dict(out_dtype=4), BAD),
    ("wgrad_fp8", dict(accumulate=2), BAD), ("wgrad_fp8", dict(lddy=7), BAD), ("wgrad_fp8", dict(dW=None), BAD),
    ("wgrad_fp8", dict(X=None), BAD), ("wgrad_fp8", dict(k=300, ld_x_scale=2), BAD),
    ("quantize_fp8", dict(X=P + 1), ALIGNMENT), ("quantize_fp8", dict(X=P + 2, dtype=1), ALIGNMENT),
    ("rmsnorm_fp8", dict(X=P + 1), ALIGNMENT), ("rmsnorm_fp8", dict(weight=P + 1), ALIGNMENT), ("rmsnorm_fp8", dict(rstd=P + 2), ALIGNMENT),
    ("rmsnorm_fp8", dict(residual=P, H=P + 1), ALIGNMENT), ("rmsnorm_fp8_backward", dict(dX=P + 1), ALIGNMENT),
    ("rmsnorm_fp8_backward", dict(dweight=P + 2), ALIGNMENT), ("rmsnorm_fp8_backward", dict(dres=P + 1), ALIGNMENT),
    ("gemm_fp8", dict(C=P + 1), ALIGNMENT), ("gemm_fp8", dict(C=P + 2, dtype=1), ALIGNMENT), ("wgrad_fp8", dict(dY=P + 1), ALIGNMENT),
    ("wgrad_fp8", dict(dW=P + 2, out_dtype=1), ALIGNMENT),
])
def test_bad_arguments(name, fields, code):
    assert _call(name, **{**_good(name), **fields}) == code
    assert vk.last_error().startswith("vk_" + name)


@pytest.mark.parametrize("name,fields", [
    ("quantize_fp8", dict(rows=0, X=None)), ("quantize_fp8", dict(cols=0, X=None)), ("rmsnorm_fp8", dict(rows=0, X=None)),
    ("gemm_fp8", dict(m=0, A=None)), ("gemm_fp8", dict(n=0, C=None)), ("wgrad_fp8", dict(n=0)), ("wgrad_fp8", dict(k=0)),
])
def test_nothing_to_do(name, fields):
    assert _call(name, **{**_good(name), **fields}) == vk.VK_OK


@pytest.mark.parametrize("name", NAMES)
def test_no_device_is_an_error(name):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert _call(name, **_good(name)) in (vk.VK_ERR_CUDA, vk.VK_ERR_NO_DEVICE)


def test_workspace_size():
    n = ctypes.c_size_t(0)
    for rows, cols in ((0, 8), (1, 1), (300, 4096), (8192, 8192)):
        assert vk.lib.vk_rmsnorm_fp8_workspace(rows, cols, ctypes.byref(n)) == vk.VK_OK
        assert rows == 0 or n.value >= 4 * cols
    assert vk.lib.vk_rmsnorm_fp8_workspace(4, 0, ctypes.byref(n)) == BAD
    assert vk.lib.vk_rmsnorm_fp8_workspace(4, 8, None) == BAD


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    w = torch.zeros(128, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.float8_e8m0fnu)
    for call in (lambda: vk.quantize_fp8(x), lambda: vk.rmsnorm_fp8(x, w), lambda: vk.gemm_fp8(q, s, q, s, trans_b=True),
                 lambda: vk.rmsnorm_fp8_backward(x, x, w, torch.zeros(4)), lambda: vk.wgrad_fp8(x, q, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        vk.quantize_fp8(x.double())
    with pytest.raises(TypeError):
        vk.rmsnorm_fp8(x.float(), w)


def test_structures_match_the_header(tmp_path):
    """Sizes and offsets of every argument structure, from the header through a C compiler."""
    pairs = {"vk_quantize_fp8_args": vk.QuantizeFp8Args, "vk_rmsnorm_fp8_args": vk.RmsnormFp8Args,
             "vk_rmsnorm_fp8_backward_args": vk.RmsnormFp8BackwardArgs, "vk_gemm_fp8_args": vk.GemmFp8Args,
             "vk_wgrad_fp8_args": vk.WgradFp8Args}
    body = "".join(f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", offsetof({c}, {f}));' for f, _ in py._fields_)
                   for c, py in pairs.items())
    src = tmp_path / "sizes.c"
    src.write_text(f'#include <stdio.h>\n#include "vkgemm.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for py in pairs.values() for v in [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]]
    assert got == want


def test_packed_arguments_match_the_structures():
    """The Python calls pack their arguments with struct formats: the same size and offsets as the structures."""
    import struct
    for name, fmt in vk._FP8_STRUCTS.items():
        cls = {"quantize_fp8": vk.QuantizeFp8Args, "rmsnorm_fp8": vk.RmsnormFp8Args, "gemm_fp8": vk.GemmFp8Args,
               "rmsnorm_fp8_backward": vk.RmsnormFp8BackwardArgs, "wgrad_fp8": vk.WgradFp8Args}[name]
        assert struct.calcsize(fmt) == ctypes.sizeof(cls), name
        fields = [f for f, _ in cls._fields_]
        got = cls.from_buffer_copy(struct.pack(fmt, *range(1, len(fields) + 1)))
        assert [getattr(got, f) for f in fields] == list(range(1, len(fields) + 1)), name


def test_oracle_form_agrees_with_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(fp8.E4M3, codes.view(torch.float8_e4m3fn).double().numpy())
    np.testing.assert_array_equal(fp8.E8M0, codes.view(torch.float8_e8m0fnu).double().numpy())
    rng = np.random.default_rng(0)
    v = np.concatenate([rng.uniform(-448, 448, 4000), rng.uniform(-0.02, 0.02, 4000), fp8.POSITIVE[:127],
                        (fp8.POSITIVE[:126] + fp8.POSITIVE[1:127]) / 2]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(fp8.round_e4m3(v.astype(np.float64)), want)


def test_oracle_scales():
    v = np.zeros((1, 128 * 6))
    for b, top in enumerate((448.0, np.nextafter(448.0, 500), 1.75, 1e-40, 0.0, np.inf)):
        v[0, 128 * b + b] = -top if b % 2 else top
    codes, s = fp8.quantize(v)
    assert s.tolist() == [[127, 128, 119, 0, 127, 255]]
    assert codes[0, 0] == 126 and (codes[0, 640:] == 127).all()
    assert not re.search("nan", str(fp8.values(codes, s)[0, :640]))


def test_stream_of_another_device_is_refused():
    """Torch would switch to the stream's device, and the call would then run on another stream of its own."""
    class Tensor:
        device = torch.device("cuda", 0)

        def get_device(self):
            return 0

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0x1000

    t, st = Tensor(), Stream()
    for call in (lambda: vk.quantize_fp8(t, stream=st), lambda: vk.rmsnorm_fp8(t, t, stream=st),
                 lambda: vk.rmsnorm_fp8_backward(t, t, t, t, stream=st), lambda: vk.gemm_fp8(t, t, t, t, stream=st),
                 lambda: vk.wgrad_fp8(t, t, t, stream=st)):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            call()


def test_arrivals_in_other_ctas_have_the_clusters_scope():
    """An arrival without a scope is a release at the CTA's: it orders nothing for a waiting thread of another CTA."""
    src = os.path.join(ROOT, "task-1", "src", "vkgemm")
    for name in sorted(os.listdir(src)):
        text = open(os.path.join(src, name)).read()
        for line in re.findall(r'"[^"]*mbarrier\.arrive[^"]*shared::cluster[^"]*"', text):
            if "tcgen05" not in line:
                assert ".cluster.shared::cluster" in line, (name, line)
    # the two data-carrying arrivals, and the waits of the pair's leader on them
    for name in ("fp8_gemm.cuh", "fp8_wgrad.cuh"):
        text = open(os.path.join(src, name)).read()
        for bar in ("tempty_bar", "full_bar(r.at)" if name == "fp8_wgrad.cuh" else "sf_full_bar(sf.at)"):
            assert re.search(r"mbar_wait_pair_warp\(" + re.escape(bar), text), (name, bar)


def test_waits_that_give_up_leave_in_order():
    """What a kernel does once a bounded wait has run out, from its source (no call makes one run out on purpose): the lanes of
    a warp with warp-wide instructions decide together, a CTA keeps its barriers, and it settles before it leaves."""
    src = os.path.join(ROOT, "task-1", "src", "vkgemm")
    for name in ("fp8_gemm.cuh", "fp8_wgrad.cuh", "fp8_thin.cuh"):
        text = open(os.path.join(src, name)).read()
        body = text[text.index("__global__"):]
        # waits by single threads: only in the loading warp's one lane
        single = re.findall(r"mbar_wait\((\w+)_bar", body)
        assert single and set(single) == {"empty"}, (name, single)
        # each role that can give up says so, and the CTA's last warp looks behind the last barrier
        assert body.count("*gave_up = 1;") == 4, name
        assert re.search(r"__syncthreads\(\);\s+if \(warp == 1 && \*gave_up != 0\) settle\(\);", body), name
        assert body.index("settle()") < body.index("tmem_dealloc"), name
    text = open(os.path.join(src, "fp8_rows.cuh")).read()
    body = text[text.index("rmsnorm_fp8_backward_kernel(const NormBackParams p)"):text.index("norm_weight_grad_kernel(")]
    assert "break" not in body and "return" not in body and "if (VEC && threadIdx.x == 0 && !ok) settle();" in body


@pytest.mark.parametrize("name,fields", [
    ("rmsnorm_fp8", dict(residual=2 * P, H=P, ldx=16, ldh=24)), ("rmsnorm_fp8", dict(residual=2 * P, H=2 * P, ld_residual=16, ldh=8)),
    ("rmsnorm_fp8_backward", dict(dX=P, dY=P, lddy=16)), ("rmsnorm_fp8_backward", dict(dX=2 * P, dres=2 * P, dY=P, lddx=16, ld_dres=8)),
])
def test_in_place_with_another_pitch_is_refused(name, fields):
    """Rows would be overwritten before they are read."""
    assert _call(name, **{**_good(name), **fields}) == BAD
    assert "in place" in vk.last_error()
    # one row has no pitch, and the same pitch is what the header allows: neither is refused for it
    for ok in (dict(rows=1), {k: 16 for k in fields if k.startswith("ld")} | {"ldh": 16, "lddx": 16, "lddy": 16, "ldx": 16, "ld_residual": 16, "ld_dres": 16}):
        args = {**_good(name), **fields, **ok}
        names = [f for f, _ in {"rmsnorm_fp8": vk.RmsnormFp8Args, "rmsnorm_fp8_backward": vk.RmsnormFp8BackwardArgs}[name]._fields_]
        if not torch.cuda.is_available():
            assert _call(name, **{k: v for k, v in args.items() if k in names}) in (vk.VK_ERR_CUDA, vk.VK_ERR_NO_DEVICE)
