"""The PyTorch binding (hxq_b200.torch_ops): operators registered with
fake (meta) implementations on CPU; on the GPU, results equal the C ABI's,
bit for bit, and the operators capture into CUDA graphs."""
import ctypes as C

import numpy as np
import pytest

from hxq_b200 import synth


def test_ops_registered_and_fake_shapes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    import hxq_b200.torch_ops  # noqa: F401  (registers torch.ops.hxq.*)
    for name in ("dequant", "vq_matmul", "affine_matmul"):
        assert hasattr(torch.ops.hxq, name)
    with FakeTensorMode():
        x = torch.empty((3, 5, 256), dtype=torch.bfloat16, device="cuda")
        y = torch.ops.hxq.vq_matmul(x, 1234, 96)
        assert y.shape == (3, 5, 96) and y.dtype == torch.float32
        codes = torch.empty((64, 256), dtype=torch.uint8, device="cuda")
        s = torch.empty((64, 2), dtype=torch.float32, device="cuda")
        y = torch.ops.hxq.affine_matmul(x, codes, s, s, None, 128)
        assert y.shape == (3, 5, 64)
        w = torch.ops.hxq.dequant(1234, 96, 256, torch.bfloat16)
        assert w.shape == (96, 256) and w.dtype == torch.bfloat16


@pytest.mark.gpu
def test_linear_and_ops_match_the_c_abi(H, L, cuda):
    torch = cuda
    from hxq_b200.torch_ops import HxqLinear
    d = synth.vq12(384, 1024, 17)
    lin = HxqLinear(d, 128, 384)
    assert lin.fused and lin.out_features == 256
    xh, _ = synth.activations(6, 1024, 18)
    x = torch.from_numpy(xh.view(np.int16)).cuda().view(torch.bfloat16).view(2, 3, 1024)
    y = lin(x)
    ref = torch.empty((6, 256), dtype=torch.float32, device="cuda")
    assert L.hxq_cuda_vq_matmul(lin.image, x.data_ptr(), 6, ref.data_ptr(), 256, None) == 0
    torch.cuda.synchronize()
    assert y.shape == (2, 3, 256)
    assert torch.equal(y.reshape(6, 256).view(torch.int32), ref.view(torch.int32))
    # weights: the decompress path, as hxq_cuda_decompress_images
    w = lin.weight(torch.float32)
    w_ref = torch.empty(256 * 1024, dtype=torch.float32, device="cuda")
    imgs = (C.c_void_p * 1)(lin.image)
    offs = (C.c_size_t * 1)(0)
    assert L.hxq_cuda_decompress_images(imgs, 1, w_ref.data_ptr(), offs, H.HXQ_OUT_F32, None, None, None) == 0
    assert L.hxq_cuda_stream_synchronize(None) == 0
    assert torch.equal(w.reshape(-1).view(torch.int32), w_ref.view(torch.int32))
    assert lin.confidence >= 0.0
    # captured into a CUDA graph on a side stream
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2 = lin(x)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y3 = lin(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y3.view(torch.int32), y.view(torch.int32)) and torch.equal(y2, y)


@pytest.mark.gpu
def test_affine_op_matches_the_c_abi(H, L, cuda):
    torch = cuda
    import hxq_b200.torch_ops  # noqa: F401
    d = synth.affine(192, 512, 128, 5, bias=True)
    codes = torch.from_numpy(d["codes"].reshape(192, 512)).cuda()
    sc = torch.from_numpy(d["scales"].reshape(192, 4)).cuda()
    of = torch.from_numpy(d["offsets"].reshape(192, 4)).cuda()
    b = torch.from_numpy(d["bias"]).cuda()
    for N in (1, 7):
        xh, _ = synth.activations(N, 512, 9)
        x = torch.from_numpy(xh.view(np.int16)).cuda().view(torch.bfloat16)
        y = torch.ops.hxq.affine_matmul(x, codes, sc, of, b, 128)
        ref = torch.empty((N, 192), dtype=torch.float32, device="cuda")
        t = H.AffineTensor(codes.data_ptr(), sc.data_ptr(), of.data_ptr(), b.data_ptr(), 192, 512, 128)
        assert L.hxq_affine_group_matmul_bf16(x.data_ptr(), C.byref(t), ref.data_ptr(), N, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int32), ref.view(torch.int32))


def test_serving_ops_fake_shapes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    import hxq_b200.torch_ops  # noqa: F401
    with FakeTensorMode():
        i = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
        q = torch.empty((7, 8, 128), dtype=torch.bfloat16, device="cuda")
        c, s = torch.empty((4, 2, 16, 128), dtype=torch.int8, device="cuda"), torch.empty((4, 2), device="cuda")
        o = torch.ops.hxq.kv_attention(q, c, c, s, s, i(4), i(3), i(3, 5), 4, 0.1, 0, True)
        assert o.shape == q.shape and o.dtype == q.dtype
        starts, lens, slots, pos, taken = torch.ops.hxq.kv_plan(i(3), i(3), i(3, 5), i(9), 16, 20)
        assert (starts.shape[0], lens.shape[0], slots.shape[0], pos.shape[0], taken.shape[0]) == (4, 3, 20, 20, 1)
        y, x = torch.empty((7, 32), device="cuda"), torch.empty((7, 64), dtype=torch.bfloat16, device="cuda")
        a, b = (torch.empty(n, dtype=torch.bfloat16, device="cuda") for n in ((2, 8, 64), (2, 32, 8)))
        assert torch.ops.hxq.lora(y, x, a, b, torch.empty(2, device="cuda"), i(4), i(3)).shape == y.shape


@pytest.mark.gpu
def test_serving_ops_match_the_calls(H, L, cuda):
    torch = cuda
    import hxq_b200.torch_ops  # noqa: F401
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    starts, lens, slots, _, _ = torch.ops.hxq.kv_plan(i(20, 3), i(0, 0), table, i(4, 2, 5, 0), 16, 23)
    one, two = S.KvCache.allocate(6, 2, 64), S.KvCache.allocate(6, 2, 64)
    k, v = torch.randn((2, 23, 2, 64), device="cuda")
    torch.ops.hxq.kv_append(one.k, one.v, one.k_scales, one.v_scales, k, v, slots)
    two.append(k, v, slots)
    assert torch.equal(one.k, two.k) and torch.equal(one.v_scales, two.v_scales)
    q = torch.randn((23, 4, 64), device="cuda").to(torch.bfloat16)
    o = torch.ops.hxq.kv_attention(q, one.k, one.v, one.k_scales, one.v_scales, starts, lens, table, 20, 0.125, 0, True)
    assert torch.equal(o, two.attention(q, starts, lens, table, 20))
    y, x = torch.randn((23, 32), device="cuda"), torch.randn((23, 64), device="cuda").to(torch.bfloat16)
    a, b = torch.randn((1, 8, 64), device="cuda").to(torch.bfloat16), torch.randn((1, 32, 8), device="cuda").to(torch.bfloat16)
    s = torch.ones(1, device="cuda")
    got = torch.ops.hxq.lora(y, x, a, b, s, starts, i(0, -1))
    assert torch.equal(got, S.LoraAdapters(a, b, s).add(y, x, S.lora_plan(starts, i(0, -1), 1, 23)))
    assert torch.equal(got[20:], y[20:]) and not torch.equal(got[:20], y[:20])


@pytest.mark.gpu
@pytest.mark.parametrize("starts,new", [([0, 4, 9], 5), ([0], 1), ([0, 0, 0], 1), ([3, 80, 150], 80)])
def test_serving_ops_rows_of_no_request(H, L, cuda, starts, new):
    """A padded step: an operator's result is its own memory, so rows that no
    request covers are defined too, whatever the allocator held before."""
    torch = cuda
    import hxq_b200.torch_ops  # noqa: F401
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    T, B = 160, len(starts) - 1
    c = S.KvCache.allocate(12, 2, 64)
    k = torch.randn((192, 2, 64), device="cuda")
    c.append(k, k.flip(0), torch.arange(192, dtype=torch.int32, device="cuda"))
    lens, table = i(*[96] * B), torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)[:B].contiguous()
    q, y = torch.randn((T, 4, 64), device="cuda").to(torch.bfloat16), torch.randn((T, 32), device="cuda")
    x = torch.randn((T, 64), device="cuda").to(torch.bfloat16)
    a, b = torch.randn((2, 8, 64), device="cuda").to(torch.bfloat16), torch.randn((2, 32, 8), device="cuda").to(torch.bfloat16)
    none = torch.ones(T, dtype=torch.bool, device="cuda")
    none[starts[0]:starts[-1]] = False
    s = torch.ones(2, device="cuda")
    for _ in range(3):   # what the allocator hands out again
        del_me = [torch.full((T, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda"), torch.full((T, 32), float("nan"), device="cuda")]
        del del_me
        o = torch.ops.hxq.kv_attention(q, c.k, c.v, c.k_scales, c.v_scales, i(*starts), lens, table, new, 0.125, 0, True)
        assert bool(o.isfinite().all()) and bool((o[none] == 0).all()) and bool((o[~none] != 0).any(-1).all())
        for yy in (y, y.t().contiguous().t()):
            got = torch.ops.hxq.lora(yy, x, a, b, s, i(*starts), i(*range(B)))
            assert torch.equal(got[none], y[none]) and bool(got.isfinite().all()) and bool((got[~none] != y[~none]).any(-1).all())
            assert got.data_ptr() != yy.data_ptr()


def test_makefile_builds_the_binding_against_pytorch_with_cuda(tmp_path):
    import os
    import subprocess

    from conftest import PKG
    torch_dir, out = tmp_path / "torch", tmp_path / "out"
    (torch_dir / "lib").mkdir(parents=True)
    out.mkdir()
    (torch_dir / "version.py").write_text("cuda = None")

    def plan():
        r = subprocess.run(["make", "-n", "-C", PKG, f"TORCH={torch_dir}", f"PYDIR={out}"], capture_output=True, text=True, check=True)
        return str(out / "_serving.so") in r.stdout
    assert not plan()                                    # a PyTorch without CUDA: the C library alone
    (torch_dir / "lib" / "libc10_cuda.so").touch()
    assert plan()
    (out / "_serving.so").touch()
    assert not plan()
    later = os.stat(out / "_serving.so").st_mtime + 10
    os.utime(torch_dir / "version.py", (later, later))   # another PyTorch
    assert plan()
