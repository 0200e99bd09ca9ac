"""`torch.ops.tessiq.<name>`: the reference's custom-operation schemas (csrc/custom_ops/*/*.cpp)
over this library's kernels, on CUDA tensors. A decline by a kernel runs the operation's ATen
definition on the same GPU, the way the reference's `call.decline` runs its `.reference()`."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import tessiq0  # noqa: E402


@pytest.fixture(scope="module")
def tessiq():
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from tessiq_b200 import ops

    ops.register_custom_ops()
    ops.register_custom_ops()          # a second call is a no-op
    return torch.ops.tessiq


def test_every_custom_operation_matches_the_oracle(tessiq):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 512, generator=g)
    w, b = 1 + torch.randn(512, generator=g) * 0.1, torch.randn(512, generator=g) * 0.1
    xd, wd, bd = x.cuda(), w.cuda(), b.cuda()
    torch.testing.assert_close(tessiq.softmax(xd, -1, False).cpu(), tessiq0.softmax(x, -1), rtol=1e-5, atol=1e-7)
    torch.testing.assert_close(tessiq.layer_norm(xd, wd, bd, 1e-5).cpu(), tessiq0.native_layer_norm(x, [512], w, b, 1e-5)[0], rtol=1e-5, atol=2e-5)
    torch.testing.assert_close(tessiq.rms_norm(xd, wd, 1e-6).cpu(), tessiq0.rms_norm(x, w, 1e-6), rtol=1e-5, atol=2e-5)
    torch.testing.assert_close(tessiq.fast_gelu(xd).cpu(), tessiq0.elementwise("fast_gelu", x), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(tessiq.swiglu(xd, xd * 0.5).cpu(), tessiq0.elementwise("swiglu", x, x * 0.5), rtol=1e-5, atol=1e-6)
    # the GEMM operations in bf16: the tensor-core kernel
    a16 = (torch.randn(96, 64, generator=g) * 0.5).bfloat16()
    w16 = (torch.randn(80, 64, generator=g) * 0.5).bfloat16()
    b16 = (torch.randn(80, generator=g) * 0.5).bfloat16()
    for name, ref in (("gemm_bias_gelu_tanh", tessiq0.gemm_bias_gelu_tanh), ("gemm_bias_gelu", tessiq0.gemm_bias_gelu)):
        expected = ref(a16, w16, b16).float()
        got = getattr(tessiq, name)(a16.cuda(), w16.cuda(), b16.cuda()).cpu().float()
        torch.testing.assert_close(got, expected, rtol=1e-2, atol=1e-2 * expected.abs().max().item())
    q, k, v = (torch.randn(1, 2, 160, 64, generator=g).bfloat16() for _ in range(3))
    expected = tessiq0.attention(q, k, v, 0.125, True).float()
    got = tessiq.attention(q.cuda(), k.cuda(), v.cuda(), 0.125, True).cpu().float()
    torch.testing.assert_close(got, expected, rtol=1e-2, atol=1e-2 * expected.abs().max().item())


def test_a_declined_call_runs_the_aten_definition_on_the_gpu(tessiq):
    # the reference's gemm_bias_gelu_tanh is an f32 operation; the tensor-core kernel declines f32
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(40, 24, generator=g), torch.randn(16, 24, generator=g), torch.randn(16, generator=g)
    got = tessiq.gemm_bias_gelu_tanh(x.cuda(), w.cuda(), b.cuda())
    assert got.is_cuda and got.dtype == torch.float32
    torch.testing.assert_close(got.cpu(), tessiq0.gemm_bias_gelu_tanh(x, w, b), rtol=1e-4, atol=1e-5)
    # pointers that are only 4-byte aligned (tests/python/test_gemm_bias_gelu_tanh.py:129-139 of the reference)
    a16 = (torch.randn(32, 64, generator=g) * 0.5).bfloat16()
    w16 = (torch.randn(48, 64, generator=g) * 0.5).bfloat16()
    b16 = torch.randn(48, generator=g).bfloat16()
    shifted = torch.empty(32 * 64 + 2, dtype=torch.bfloat16, device="cuda")[2:].view(32, 64)
    shifted.copy_(a16)
    assert shifted.data_ptr() % 16 == 4
    expected = tessiq0.gemm_bias_gelu_tanh(a16, w16, b16).float()
    got = tessiq.gemm_bias_gelu_tanh(shifted, w16.cuda(), b16.cuda()).cpu().float()
    torch.testing.assert_close(got, expected, rtol=1e-2, atol=1e-2 * expected.abs().max().item())
    # heads of 256: no attention kernel
    q = torch.randn(1, 2, 64, 256, generator=g).bfloat16()
    expected = tessiq0.attention(q, q, q, 256 ** -0.5, False).float()
    got = tessiq.attention(q.cuda(), q.cuda(), q.cuda(), 256 ** -0.5, False).cpu().float()
    torch.testing.assert_close(got, expected, rtol=2e-2, atol=2e-2 * expected.abs().max().item())


def test_host_tensors_have_no_implementation(tessiq):
    with pytest.raises((NotImplementedError, RuntimeError)):
        tessiq.fast_gelu(torch.randn(8))


def test_window_attention_and_the_cache_are_operations_too(tessiq):
    from tessiq_b200 import ops

    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, n, t, 64, generator=g).bfloat16().cuda() for n, t in ((4, 5), (2, 40), (2, 40)))
    assert torch.equal(tessiq.window_attention(q, k, v, 16, 2, None), ops.window_attention(q, k, v, 16, 2))
    # f32 has no kernel: the ATen definition, queries before the first key included
    wide = tessiq.window_attention(q.float(), k.float()[:, :, :3], v.float()[:, :, :3], None, 0, 0.1)
    assert wide.dtype == torch.float32 and wide[:, :, :2].count_nonzero().item() == 0
    narrow = ops.window_attention(q, k[:, :, :3].contiguous(), v[:, :, :3].contiguous(), scale=0.1)
    # (bf16 against f32: half a step of the result, 2^-8, and at most as much of the weights)
    torch.testing.assert_close(narrow.float(), wide, rtol=2.0**-7, atol=2.0**-7 * v.float().abs().max().item())
    pages = [torch.zeros(6, 2, 16, 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(6, 2, device="cuda") for _ in range(2)]
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32).cuda()
    starts, lengths = torch.zeros(2, dtype=torch.int32).cuda(), torch.tensor([40, 30], dtype=torch.int32).cuda()
    tessiq.cache_store(k, v, *pages, *scales, table, starts, lengths)
    got = tessiq.cache_attention(q, *pages, *scales, table, lengths, 16, 2, None)
    assert torch.equal(got, ops.cache_attention(q, *pages, *scales, table, lengths, 16, 2)) and got.isfinite().all()
    tessiq.copy_pages([*(p.view(torch.uint8) for p in pages), *scales], [0], [5], 0)
    assert torch.equal(scales[0][5], scales[0][0]) and torch.equal(pages[1].view(torch.uint8)[5], pages[1].view(torch.uint8)[0])


def test_window_attention_that_has_no_kernel_is_in_f32_or_f64_and_keeps_hidden_keys_out(tessiq):
    from test_cache import by_rows, roundings

    g = torch.Generator().manual_seed(3)
    for dtype, width in ((torch.float64, 64), (torch.float32, 64), (torch.bfloat16, 256)):
        q, k, v = (torch.randn(1, n, t, width, generator=g).to(dtype) for n, t in ((4, 3), (2, 40), (2, 40)))
        k[:, :, 10:20], v[:, :, 10:20] = float("nan"), float("inf")      # between the sinks and the first query's window
        got = tessiq.window_attention(q.cuda(), k.cuda(), v.cuda(), 16, 4, None)
        exact = by_rows(q, k, v, 16, 4, width**-0.5)
        assert got.dtype == dtype and got.isfinite().all()
        inside = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2
        assert ((got.cpu().double() - exact).abs() <= torch.finfo(dtype).eps / 2 * exact.abs() + inside * roundings(q, k, v, width**-0.5)).all()
