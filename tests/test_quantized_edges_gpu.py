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


def step_context(T, dtype, **options):
    """A StepContext as far as products and gated units look at it."""
    from rocmforge_b200.engine.context import Options, StepContext
    ctx = object.__new__(StepContext)
    ctx.options, ctx.compute_dtype, ctx.T = Options(weight_bits=4, **options), dtype, T
    return ctx


def unit(activation, g, u):
    if activation == "clamped_glu":
        g, u = g.clamp_max(3), u.clamp(-3, 3)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return dict(silu=lambda: g * torch.sigmoid(g), relu=lambda: g.clamp_min(0),
                gelu_tanh=lambda: g / (1 + torch.exp(-2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))))[activation]() * u


@pytest.mark.parametrize("row_bits", [8, 16])
@pytest.mark.parametrize("activation", ["silu", "relu", "gelu_tanh", "clamped_glu"])
@pytest.mark.parametrize("T", [1, 5, 32, 40, 300, 600])
def test_the_unit_is_formed_from_32_bit_sums(T, activation, row_bits):
    """Gate and up are whole numbers of 2^-10, exact in 32 bits and not in 16; the unit of them is rounded once, to the rows' dtype or to 8 bits."""
    from rocmforge_b200 import kernels
    from rocmforge_b200.parts.linear import Linear
    K, I, G = 256, 136, 64
    gen = torch.Generator().manual_seed(T)
    q = torch.randint(-8, 8, (2 * I, K), generator=gen, dtype=torch.int8)
    w = kernels.W4Weight.from_quantized(q.to(DEV), torch.full((2 * I, K // G), 2.0 ** -10, device=DEV), G)
    x = torch.randint(-8, 9, (T, K), generator=gen).to(BF).to(DEV)
    gu = (x.double() @ q.to(DEV).double().T / 1024).cpu()
    want = unit(activation, gu[:, ::2], gu[:, 1::2])
    linear = object.__new__(Linear)
    linear.weight, linear.bias, linear.N, linear.K = w, None, 2 * I, K
    ctx = step_context(T, BF, row_bits=row_bits)
    # whole numbers in 8 bits: the scale of a group is its largest / 127, so the rows are made by hand
    y = x
    if row_bits == 8 and T <= 32:
        full = torch.zeros(T, K, dtype=torch.int8, device=DEV)
        full[:] = x.to(torch.int8)
        y = kernels.Q8Rows(full, torch.ones(T, K // G, device=DEV), K, G, BF)
    kw = dict(limit=3.0, alpha=1.702) if activation == "clamped_glu" else {}
    got = ctx.gated_activation(y, linear, activation, reader=w, **kw)
    assert got.dtype == BF and tuple(got.shape) == (T, I)
    # the unit in 32 bits: an argument of at most 25 off by seven roundings, an exponential by two units, three more roundings; 1 + u rounds as well
    rel = (7 * 25 + 8) * 2.0 ** -24
    if isinstance(got, kernels.Q8Rows):
        check_rows(got, want, rel)
    else:
        got = got.cpu().double()
        bound = (2.0 ** -8 + 2 * rel) * want.abs() + 1e-30
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("activation", ["silu", "relu", "gelu_tanh", "clamped_glu"])
@pytest.mark.parametrize("T,I,off", [(0, 8, 0), (1, 1, 0), (3, 101, 0), (7, 64, 1), (130, 1000, 2), (700, 640, 0)])
def test_units_of_32_bit_sums_rounded_once(activation, T, I, off):
    """``swiglu`` and ``clamped_glu`` with a result in bfloat16 from float32, on any boundary."""
    from rocmforge_b200 import kernels
    memory = torch.zeros(2 * T * I + 4, device=DEV)
    gu = memory[off:off + 2 * T * I].view(T, 2 * I)
    gu.copy_(2 * numbers(T, 2 * I, spread=False))
    want = unit(activation, gu.cpu().double()[:, ::2], gu.cpu().double()[:, 1::2])
    got = (kernels.clamped_glu(gu, 3.0, 1.702, dtype=BF) if activation == "clamped_glu" else kernels.swiglu(gu, activation=activation, dtype=BF))
    assert got.dtype == BF and got.shape == (T, I)
    # the exponential's argument: seven roundings of at most 80 where the exponential is not yet 2^-110 (what is left there is below 2^-100)
    bound = (2.0 ** -8 + (7 * 80 + 8) * 2.0 ** -24) * want.abs() + 2.0 ** -100
    assert ((got.cpu().double() - want).abs() <= bound).all()
    with pytest.raises(kernels.KernelError):
        kernels.swiglu(gu.to(BF), dtype=F32)
    with pytest.raises(kernels.KernelError):
        kernels.clamped_glu(gu.to(BF), 3.0, 1.0, dtype=F32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["D", "FA", "FC", "FD", "RA"])
def test_weight_bytes_are_what_the_products_hold(folders, name, dtype):
    """Zero rows that a part adds to a fused weight lie on the device too, in 16 bits as in 4 (FA, FC and FD have some)."""
    import rocmforge_b200 as rf
    from rocmforge_b200 import kernels
    from rocmforge_b200.weights.loader import load_folder
    from test_quantized_engine_gpu import TORCH
    for bits in (16, 4):
        m = rf.Model.from_folder(folders(name, dtype), dtype=TORCH[dtype], options=rf.Options(weight_bits=bits, weight_group=32))
        params = load_folder(folders(name, dtype), m.spec.param_specs(), TORCH[dtype], "cpu")
        others, held = {}, 0                             # (tied tensors count once)
        for prefix, part in m.spec.named_parts().items():
            for local, spec in part.param_specs().items():
                if not (part.linears() and spec.kind == "matrix") and prefix + local in params:
                    others[params[prefix + local].data_ptr()] = params[prefix + local].nbytes
            for linear in part.linears():
                assert isinstance(linear.weight, kernels.W4Weight) == (bits == 4)
                held += linear.weight.nbytes
        assert m.weight_bytes == held + sum(others.values())


@pytest.mark.parametrize("tied", [False, True])
def test_a_model_in_4_bits_never_lies_on_the_device_in_16(tmp_path, tied):
    """Loaded part after part: the most memory that is held at once is the 4-bit model and one part in 16 bits (with its fused copy)."""
    import rocmforge_b200 as rf
    from helpers import CONFIGS, write_tiny
    cfg = dict(CONFIGS["D"], num_hidden_layers=12, hidden_size=512, intermediate_size=2048, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
               tie_word_embeddings=tied)
    write_tiny(cfg, str(tmp_path), "bfloat16")
    make = lambda bits: rf.Model.from_folder(str(tmp_path), options=rf.Options(weight_bits=bits))  # noqa: E731
    sixteen = make(16).weight_bytes
    m = make(4)                                          # (everything is built and allocated that stays)
    m.new_cache(max_tokens=64)
    four = m.weight_bytes
    del m
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    m = make(4)
    held, peak = torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before
    part = 2 * 3 * 512 * 2048                            # the feed-forward, the largest part: its tensors, two of them fused once more
    assert four <= held <= four + 2 ** 20 and peak <= four + 2 * part + 2 ** 20 and peak < 0.6 * sixteen


# ---------------------------------------------------------------- sums of whole numbers, exact in 32 bits in whatever order
def whole(kind, M, N, K, G, seed=0):
    """Rows, a weight and the product, all whole numbers (scales are 1), every partial sum below 2^24."""
    from rocmforge_b200 import kernels
    gen = torch.Generator().manual_seed(seed + M + N + K)
    q = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(DEV)
    x = torch.randint(-9, 10, (M, K), generator=gen, dtype=torch.int8).to(DEV)
    assert 9 * 8 * K < 2 ** 24
    w = kernels.W4Weight.from_quantized(q, torch.ones(N, (K + G - 1) // G, device=DEV), G)
    want = (x.double() @ q.double().T).float()
    if kind != "q8":
        return x.to(BF if kind == "bf16" else F32), w, want
    Kp = kernels.padded_columns(K, G)
    full = torch.zeros(M, Kp, dtype=torch.int8, device=DEV)
    full[:, :K] = x
    return kernels.Q8Rows(full, torch.ones(M, Kp // G, device=DEV), K, G, BF), w, want


@pytest.mark.parametrize("kind", ["q8", "bf16", "f32"])
@pytest.mark.parametrize("M", [1, 5, 16, 31, 64, 130, 530])
@pytest.mark.parametrize("N,K,G", [(48, 19001, 32), (130, 19008, 64), (200, 18944, 128), (1003, 1100, 32), (17, 65, 128)])
def test_every_column_counts_once(kind, M, N, K, G):
    """Equal to the last bit: a column left out or counted twice, or a number in the wrong place, shows at any length."""
    from rocmforge_b200 import kernels
    x, w, want = whole(kind, M, N, K, G)
    b, h = torch.arange(N, device=DEV, dtype=F32) - 7, torch.arange(M * N, device=DEV, dtype=F32).view(M, N) % 1000
    assert torch.equal(kernels.gemm_w4(x, w, b, out_f32=True), want + b)
    assert torch.equal(kernels.gemm_w4(x, w, out=h.clone(), accumulate=True), want + h)
    assert torch.equal(kernels.gemm_w4(x, w), want if kind == "f32" else want.to(BF))
    assert torch.equal(kernels.gemm_w4(x, w, b, out_f32=True, tensor_cores=False), want + b)


@pytest.mark.parametrize("splits", [1, 2, 5, 8])
@pytest.mark.parametrize("kind,plan", [("q8", (1, 1, 1)), ("q8", (1, 1, 16)), ("q8", (2, 1, 4)), ("q8", (2, 2, 2)), ("q8", (4, 1, 8)), ("q8", (4, 2, 4)),
                                       ("bf16", (1, 1, 1)), ("bf16", (1, 1, 8)), ("bf16", (2, 1, 2)), ("bf16", (2, 2, 4)), ("bf16", (32,)), ("bf16", (64,)), ("bf16", (128,))])
def test_every_column_counts_once_in_every_plan(monkeypatch, kind, plan, splits):
    from rocmforge_b200 import kernels
    from rocmforge_b200.kernels import quantized
    for M, N, K, G in ((33, 300, 4228, 32), (8, 96, 2050, 64), (17, 450, 6400, 128)):
        clusters = 3
        monkeypatch.setattr(quantized, "w4_launch", lambda *a: (*plan, splits) if len(plan) == 1 else (*plan, splits, clusters))
        if len(plan) == 3:
            fits = quantized._f("rf_gemm_w4_shared")(0 if kind == "q8" else 1, M, N, K, G, *plan, splits, clusters) <= quantized.W4_MOST_SHARED
            if not fits:
                continue
        x, w, want = whole(kind, M, N, K, G)
        h = torch.arange(M * N, device=DEV, dtype=F32).view(M, N) % 1000
        assert torch.equal(kernels.gemm_w4(x, w, out=h.clone(), accumulate=True), want + h)
        assert torch.equal(kernels.gemm_w4(x, w), want.to(BF))


# ---------------------------------------------------------------- the engine
@pytest.mark.parametrize("row_bits", [8, 16])
def test_sequences_go_on_alike_in_graphs_and_out_of_them(folders, row_bits):
    """Decode graphs of one, two and three sequences, replayed in turn with steps outside graphs between them: token by token what the same
    batches give without any graph."""
    import rocmforge_b200 as rf
    from helpers import random_tokens
    make = lambda graphs: rf.LLM(folders("D", "bfloat16"), options=rf.Options(weight_bits=4, weight_group=64, row_bits=row_bits, decode_graphs=graphs))  # noqa: E731
    graphs, plain = make(True), make(False)
    prompts = [random_tokens(300, n, n) for n in (40, 21, 33)]
    for batch in (prompts[:1], prompts[:2], prompts, prompts[1:], prompts[:2], prompts[:1]):
        runner = graphs.engine and graphs.engine.decode_runner
        before = runner.replays if runner else 0
        got = [r.tokens for r in graphs.generate(batch, max_tokens=12, temperature=0.0, stop_token_ids=[])]
        assert graphs.engine.decode_runner.replays > (before if graphs.engine.decode_runner is runner else 0)
        want = [r.tokens for r in plain.generate(batch, max_tokens=12, temperature=0.0, stop_token_ids=[])]
        assert plain.engine.decode_runner is None and got == want and all(len(t) == 12 for t in got)


@pytest.mark.parametrize("row_bits", ["8", "16"])
def test_the_command_line_passes_its_options_on(folders, monkeypatch, row_bits):
    """The options reach the model, and the ids that the command prints are those of a model made with the same ones."""
    import os
    import subprocess
    import sys

    import rocmforge_b200 as rf
    from helpers import ROOT
    from rocmforge_b200 import cli, kernels
    from rocmforge_b200.engine import model
    seen, real = [], model.Model.__init__

    def init(self, *a, **kw):
        real(self, *a, **kw)
        seen.append(self)
    argv = ["--model", folders("D", "bfloat16"), "--prompt-ids", "1,2,3,4,5", "--max-tokens", "8", "--temperature", "0", "--stop-ids", "",
            "--weight-bits", "4", "--weight-group", "32", "--row-bits", row_bits]
    monkeypatch.setattr(model.Model, "__init__", init)
    assert cli.main(argv) == 0
    options = seen[0].options
    assert (options.weight_bits, options.weight_group, options.row_bits) == (4, 32, int(row_bits))
    assert all(isinstance(a.weight, kernels.W4Weight) and a.weight.group == 32 for p in seen[0].spec.named_parts().values() for a in p.linears())
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "rocmforge"), *argv, "--debug"], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    got = [int(line.split("token_id=")[1]) for line in run.stderr.splitlines() if line.startswith("[Generated]")]
    llm = rf.LLM(folders("D", "bfloat16"), options=rf.Options(weight_bits=4, weight_group=32, row_bits=int(row_bits), decode_graphs=False))
    assert got == llm.generate([[1, 2, 3, 4, 5]], max_tokens=8, temperature=0.0, stop_token_ids=[])[0].tokens


OTHERS = ["RC", "VB", "VC", "VE", "FB", "FD", "LB", "LD", "GB", "GC", "GD", "GF", "DB", "DD"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", OTHERS)
def test_the_other_designs(folders, name, dtype):
    """The variants of each design that the engine's tests of 4-bit weights leave out, by the same bounds."""
    from helpers import random_tokens
    from test_quantized_engine_gpu import assert_both_close, pair, run_both
    four, full = pair(folders, name, dtype, 32, 16)
    V = four.spec.vocab_size
    longest = min(100, four.spec.max_position - 8)
    for lens in ((5, 17), (longest, min(51, longest))):
        a, b = run_both(four, full, [random_tokens(V, n, n) for n in lens], V)
        assert_both_close(a, b, dtype, f"{name} {dtype} {lens}")


def to_8_bits(y, G, dtype):
    """``Q8Rows`` of numbers in 64 bits."""
    from rocmforge_b200 import kernels
    T, K = y.shape
    p = torch.zeros(T, kernels.padded_columns(K, G), dtype=torch.float64, device=y.device)
    p[:, :K] = y
    p = p.view(T, -1, G)
    a = p.abs().amax(-1, keepdim=True) / 127
    q = torch.where(a > 0, p / a, 0.0).round().to(torch.int8)
    return kernels.Q8Rows(q.view(T, -1), a.float().view(T, -1), K, G, dtype)


def plain_gemm_w4(x, w, bias=None, *, out=None, out_f32=False, accumulate=False, tensor_cores=True):
    from rocmforge_b200 import kernels
    x64 = (x.q.double() * x.scales.double().repeat_interleave(x.group, 1))[:, :x.K] if type(x) is kernels.Q8Rows else x.double()
    y = x64 @ kernels.dequantize_w4(w, F32).double().T + (0 if bias is None else bias.double())
    return out.copy_(out.double() + y) if accumulate else y.to(F32 if out_f32 else x.dtype)


def plain_add_rmsnorm_q8(h, weight, eps, dtype, group=128, pending=None, rows=None):
    if pending is not None:
        h.add_(pending.sum(0) if pending.dim() == 3 else pending.float())
    x = h.double()
    return to_8_bits(x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double(), group, dtype)


def plain_swiglu_q8(gu, group=128, activation="silu", dtype=None):
    return to_8_bits(unit(activation, gu.double()[:, ::2], 1) * gu.double()[:, 1::2], group, dtype or gu.dtype)


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "RA", "RB", "VA", "VD", "FA", "FC", "LA", "LC", "GA", "GE", "DA", "DC", *OTHERS])
def test_8_bit_rows_in_the_engine_are_those_of_the_formulas(folders, monkeypatch, name):
    """Every design in 32 bits with 8-bit rows, against itself with the operators in 64 bits: the same numbers to 32-bit accuracy.  A number that lies
    on the border between two steps may fall to either side, which shows in the logits after it and in no others; what is wrong shows in all."""
    import rocmforge_b200 as rf
    from helpers import random_tokens
    from rocmforge_b200 import kernels
    m = rf.Model.from_folder(folders(name, "float32"), dtype=F32, options=rf.Options(weight_bits=4, weight_group=32))
    V, out, used = m.spec.vocab_size, [], set()
    for plain in (False, True):
        if plain:
            for f in (plain_gemm_w4, plain_add_rmsnorm_q8, plain_swiglu_q8):
                monkeypatch.setattr(kernels, f.__name__[6:], lambda *a, f=f, **kw: (used.add(f.__name__), f(*a, **kw))[1])
            monkeypatch.setattr(kernels, "quantize_q8", lambda x, group=128: to_8_bits(x.double(), group, x.dtype))
        cache = m.new_cache(max_tokens=64 * 24, max_slots=4)
        slots = [cache.alloc_slot() for _ in (5, 17)]
        got = [m.step(cache, [rf.StepRequest(s, p, [0, len(p) - 1]) for s, p in zip(slots, [random_tokens(V, n, n) for n in (5, 17)])])]
        for d in range(3):
            got.append(m.step(cache, [rf.StepRequest(s, [random_tokens(V, 1, 10 * d + i)[0]], [0]) for i, s in enumerate(slots)]))
        out.append(torch.cat(got).cpu().double())
    assert "plain_gemm_w4" in used
    off = (out[0] - out[1]).norm(dim=1) / out[1].norm(dim=1)
    assert torch.isfinite(out[0]).all() and int((off < 1e-5).sum()) >= 3, off
