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


@pytest.fixture
def launched(monkeypatch):
    """The names of the launchers that are called from here on."""
    from rocmforge_b200.kernels import basic, latent, layernorm, quantized, tensor_core
    names = []
    for module in (basic, quantized, tensor_core):
        for look in [n for n in ("_f", "_fc") if hasattr(module, n)]:
            def spy(*a, real=getattr(module, look)):
                names.extend(x for x in a if isinstance(x, str) and x.startswith("rf_"))
                return real(*a)
            monkeypatch.setattr(module, look, spy)
    return names


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("M,N,K", [(1, 48, 100), (20, 300, 2176), (64, 4608, 896), (200, 130, 1100), (1030, 130, 2304), (3, 40, 70016)])
def test_products_without_the_tcgen05_kernels(launched, dt, M, N, K):
    from rocmforge_b200 import kernels
    w, full = weight(N, K, 64)
    x = numbers(M, K, dt=dt).to(DEV)
    full, x64, b, h = full.to(DEV), x.double(), numbers(N, seed=2).to(DEV), numbers(M, N, seed=9).to(DEV)
    want, size = x64 @ full.T + b.double(), x64.abs() @ full.abs().T + b.double().abs()
    del launched[:]
    close(kernels.gemm_w4(x, w, b, tensor_cores=False), want, size, 2 * K + 25, dt)
    close(kernels.gemm_w4(x, w, b, out_f32=True, tensor_cores=False), want, size, 2 * K + 25, F32)
    close(kernels.gemm_w4(x, w, b, out=h.clone(), accumulate=True, tensor_cores=False), want + h.double(), size + h.double().abs(), 2 * K + 26, F32)
    assert launched and not [n for n in launched if "_tc" in n], launched


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("row_bits", [8, 16])
def test_the_engine_without_the_tcgen05_kernels(folders, launched, dtype, row_bits):
    """``Options(tensor_core_gemm=False)`` holds for products with 4-bit weights as well, in prompts of few and of many tokens and in single steps."""
    import rocmforge_b200 as rf
    from helpers import random_tokens
    from test_quantized_engine_gpu import TORCH, assert_both_close, run_both
    make = lambda on: rf.Model.from_folder(folders("D", dtype), dtype=TORCH[dtype],  # noqa: E731
                                           options=rf.Options(weight_bits=4, weight_group=32, row_bits=row_bits, tensor_core_gemm=on, tcgen05_attention=on))
    off, on = make(False), make(True)
    for lens in ((5,), (17, 100), (600,)):
        del launched[:]
        prompts = [random_tokens(off.spec.vocab_size, n, n) for n in lens]
        a, _ = run_both(off, off, prompts, off.spec.vocab_size)
        # (32-bit rows that stay what they are go by the weights written out)
        assert ("rf_dequantize_w4" if (dtype, row_bits) == ("float32", 16) else "rf_gemm_w4") in launched
        assert not [n for n in launched if "_tc" in n and "attention" not in n], sorted(set(launched))
        b, _ = run_both(on, on, prompts, on.spec.vocab_size)
        assert_both_close(a, b, dtype, f"{dtype} {lens}")


@pytest.mark.parametrize("M,K,G", [(32, 100000, 32), (32, 100000, 64), (8, 140000, 32), (9, 140001, 64), (8, 140000, 128), (1, 300000, 128)])
def test_long_8_bit_rows(M, K, G):
    from rocmforge_b200 import kernels
    N = 40
    w, full = weight(N, K, G)
    r = kernels.quantize_q8(numbers(M, K, dt=BF).to(DEV), G)
    full, x64, b, h = full.to(DEV), stands_for(r).to(DEV), numbers(N, seed=2).to(DEV), numbers(M, N, seed=9).to(DEV)
    want, size, terms = x64 @ full.T + b.double(), x64.abs() @ full.abs().T + b.double().abs(), K // 32 + 25
    close(kernels.gemm_w4(r, w, b), want, size, terms, BF)
    close(kernels.gemm_w4(r, w, b, out_f32=True), want, size, terms, F32)
    close(kernels.gemm_w4(r, w, b, out=h.clone(), accumulate=True), want + h.double(), size + h.double().abs(), terms + 1, F32)


@pytest.mark.parametrize("H", [32768, 32769, 40000])
def test_a_wide_norm_hands_on_what_it_can(H):
    """The 8-bit norm takes 32,768 columns; a part with more gets the norm's ordinary rows, and its product makes 8 bits of them."""
    from rocmforge_b200 import kernels
    from rocmforge_b200.engine.stream import ResidualStream
    from rocmforge_b200.parts.norm import RMSNorm
    norm = RMSNorm(H, 1e-6)
    norm.bind({"weight": torch.ones(H, device=DEV)}, BF)
    h, p = numbers(3, H), numbers(2, 3, H, seed=4)
    stream = ResidualStream(h.to(DEV))
    stream.add_pending(p.to(DEV))
    y = norm.forward_q8(None, stream, 64)
    new = h + p[0] + p[1]
    assert stream.pending is None and torch.equal(stream.h.cpu(), new)
    x = new.double()
    want = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    if H <= 32768:
        check_rows(y, want, 60 * 2.0 ** -24)
    else:
        assert y.dtype == BF and ((y.cpu().double() - want).abs() <= (2.0 ** -8 + 60 * 2.0 ** -24) * want.abs()).all()
        check_rows(kernels.quantize_q8(y, 64), y.cpu().double(), 0)
