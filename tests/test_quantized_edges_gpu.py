"""Edges of the 4-bit weight path on the device, against plain forms in 64 bits."""
import pytest
import torch

from test_quantized_gpu import BF, DEV, F32, check_rows, close, numbers, stands_for, weight

pytestmark = pytest.mark.gpu


def test_norm_of_rows_that_the_kernel_before_has_chosen():
    """The rows' indices come from a kernel of this library launched right before (in a graph too, where its successor starts early)."""
    from rocmforge_b200 import kernels
    T, H, G = 64, 896, 64
    h, w = numbers(T, H).to(DEV), torch.ones(H, device=DEV)
    logits = torch.zeros(200, T, device=DEV)
    ids = torch.zeros(200, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        def body():
            kernels.argmax(logits, out=ids)
            return kernels.add_rmsnorm_q8(h, w, 1e-6, BF, G, rows=ids)
        body()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = body()
        x = h.cpu().double()
        want = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        for seed in (1, 2, 3):
            logits.copy_(numbers(200, T, seed=seed))
            graph.replay()
            torch.cuda.synchronize()
            check_rows(got, want[logits.cpu().argmax(-1)], 60 * 2.0 ** -24)
            check_rows(body(), want[logits.cpu().argmax(-1)], 60 * 2.0 ** -24)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,I", [(3, 1), (40, 33), (40, 65), (9, 129), (5, 256)])
def test_gelu_of_strongly_negative_gates(dt, G, T, I):
    """Gates of -6 .. -4, where 1 + tanh has lost most of its bits: a group of nothing else gets its scale from values near 1e-8."""
    from rocmforge_b200 import kernels
    gu = numbers(T, 2 * I, spread=False)
    gu[:, ::2] = -4 - 2 * torch.rand(T, I, generator=torch.Generator().manual_seed(I))
    gu = gu.to(dt)
    g, u = gu.double()[:, ::2], gu.double()[:, 1::2]
    twice = 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)
    r = kernels.swiglu_q8(gu.to(DEV), G, activation="gelu_tanh")
    # the exponent's argument, at most 25, is off by at most seven roundings; the exponential by two units, the sum, quotient and product by a rounding each
    check_rows(r, g / (1 + torch.exp(-twice)) * u, (7 * 25 + 4 + 3) * 2.0 ** -24)


@pytest.mark.parametrize("off", [1, 2, 3, 5])
@pytest.mark.parametrize("M,N,K", [(520, 256, 512), (2100, 1024, 2304), (1100, 384, 72), (40, 256, 512), (3, 256, 512)])
def test_results_anywhere_in_memory(M, N, K, off):
    """``out`` on the boundary of its type alone, whatever the number of tokens, and what lies beside it left alone."""
    from rocmforge_b200 import kernels
    w, full = weight(N, K, 64)
    x = numbers(M, K, dt=BF).to(DEV)
    full, x64 = full.to(DEV), x.double()
    want, size, terms = x64 @ full.T, x64.abs() @ full.abs().T, 2 * K + 24
    h = numbers(M, N, seed=9).to(DEV)
    for dt, kw, more in ((BF, {}, 0), (F32, dict(out_f32=True), 0), (F32, dict(accumulate=True), 1)):
        memory = torch.full((M * N + 16,), 7.0, dtype=dt, device=DEV)
        out = memory[off:off + M * N].view(M, N)
        if more:
            out.copy_(h)
        assert kernels.gemm_w4(x, w, out=out, **kw) is out
        close(out, want + h.double() * more, size + h.double().abs() * more, terms + more, dt)
        assert (memory[:off] == 7).all() and (memory[off + M * N:] == 7).all()
    kernels.tensor_core.check_status(torch.device(DEV))
