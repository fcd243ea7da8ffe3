"""Weights in 4 bits, rows in 8 bits and the products that read them, against plain forms in 64 bits."""
import pytest
import torch

from test_quantized import unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}                  # a rounding, relative


def numbers(*shape, seed=0, dt=F32, spread=True):
    g = torch.Generator().manual_seed(seed + sum(shape))
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp(0.7 * torch.randn(shape[-1], generator=g))
    return x.to(dt)


def weight(N, K, G, seed=0):
    """A 4-bit weight and its numbers in 64 bits, scales of five significant bits."""
    from rocmforge_b200 import kernels
    g = torch.Generator().manual_seed(seed + N + K)
    q = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
    s = ((16 + torch.randint(0, 16, (N, (K + G - 1) // G), generator=g)) / 512).bfloat16()
    full = q.double() * s.double().repeat_interleave(G, 1)[:, :K]
    return kernels.W4Weight.from_quantized(q.to(DEV), s.to(DEV), G), full


def stands_for(r):
    """The numbers of Q8Rows, in 64 bits."""
    return (r.q.cpu().double() * r.scales.cpu().double().repeat_interleave(r.group, 1))[:, :r.K]


def close(got, want, size, terms, dt):
    """Sums of ``terms`` numbers of total magnitude ``size`` in 32 bits, then one rounding to ``dt``."""
    want, got = want.to(DEV), got.double()
    bound = terms * 2.0 ** -24 * size.to(DEV) + HALF[dt] * want.abs()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound.clamp_min(1e-300)).max())


# ---------------------------------------------------------------- rows
def check_rows(r, want, rel):
    """8-bit rows of numbers known to ``rel``: the scale is max / 127, every number the nearest step, padding is zero."""
    T, K = want.shape
    G, groups = r.group, r.scales.shape[1]
    full = torch.zeros(T, groups * G, dtype=torch.float64)
    full[:, :K] = want
    full = full.view(T, groups, G)
    s, q = r.scales.cpu().double(), r.q.cpu().double().view(T, groups, G)
    top = full.abs().amax(-1)
    assert ((s - top / 127).abs() <= (rel + 2.0 ** -23) * top / 127).all()
    assert (q.abs() <= 127).all() and (q[top == 0] == 0).all()
    assert ((q * s[..., None] - full).abs() <= s[..., None] * (0.5 + 127 * (rel + 2.0 ** -21))).all()
    assert not r.q[:, K:].any()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 64), (3, 100), (5, 127), (2, 1028), (70, 896), (1, 19001)])
def test_rows_to_8_bits(dt, G, T, K):
    from rocmforge_b200 import kernels
    x = numbers(T, K, dt=dt)
    x[:, :min(K, 40)] *= 0 if T == 5 else 1              # groups of zeros
    r = kernels.quantize_q8(x.to(DEV), G)
    check_rows(r, x.double(), 0)
    for d in (F32, BF):
        back = r.materialize(d)
        assert back.shape == (T, K) and torch.equal(back.cpu(), (r.q.cpu().float() * r.scales.cpu().repeat_interleave(G, 1))[:, :K].to(d))
    assert r.materialize().dtype == dt


def test_rows_any_distance_apart_and_many_of_them():
    from rocmforge_b200 import kernels
    x = numbers(9, 300)
    for cut in (x[:, 3:203], x[:, 4:204], x[::2, :128], x[:, :1]):
        check_rows(kernels.quantize_q8(x.to(DEV)[:, cut.storage_offset() % 300:][::cut.stride(0) // 300, :cut.shape[1]], 32), cut.double(), 0)
    many = numbers(70001, 8, spread=False)
    check_rows(kernels.quantize_q8(many.to(DEV), 64), many.double(), 0)
    assert kernels.quantize_q8(torch.empty(0, 64, device=DEV), 64).shape == (0, 64)


def test_groups_that_hold_no_ordinary_numbers():
    from rocmforge_b200 import kernels
    x = numbers(6, 256)
    x[0, 5], x[1, 70], x[2, 130], x[3] = float("nan"), float("inf"), -float("inf"), 0
    x[4] *= 2.0 ** -140                                  # held as zeros: below 2^-120
    x[5] *= 2.0 ** 100
    r = kernels.quantize_q8(x.to(DEV), 64)
    s = r.scales.cpu()
    nan = torch.zeros(6, 4, dtype=torch.bool)
    nan[0, 0] = nan[1, 1] = nan[2, 2] = True
    assert torch.equal(s.isnan(), nan) and not s[3:5].any() and not r.q[3:5].any()
    keep = x.clone()
    keep[0, :64] = keep[1, 64:128] = keep[2, 128:192] = keep[4] = 0
    r.scales[torch.isnan(r.scales)] = 0
    check_rows(r, keep.double(), 0)


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (17, 100), (40, 896), (130, 1100)])
def test_weights_to_4_bits_and_back(dt, G, N, K):
    from rocmforge_b200 import kernels
    x = numbers(N, K + 3, dt=dt)
    x[0, :50] = 0
    w = kernels.quantize_w4(x.to(DEV)[:, 3:], G)         # rows that start anywhere
    x = x[:, 3:]
    q, s = unpacked(w)
    assert not q[N:].any() and not q[:, K:].any() and not s[N:].any()
    q, s = q[:N, :K].double(), s[:N]
    groups = torch.zeros(N, s.shape[1] * G)
    groups[:, :K] = x.float()
    top = groups.view(N, -1, G).abs().amax(-1)
    m, e = torch.frexp(top / 7.5)
    assert torch.equal(s.float(), torch.ldexp((m * 32).round() / 32, e))            # five significant bits
    step = s.double().repeat_interleave(G, 1)[:, :K]
    off = (x.double() - q * step).abs()
    inside = x.double().abs() <= 7.5 * step
    assert (off[inside] <= (0.5 + 2.0 ** -20) * step[inside]).all() and (off <= 0.75 * step).all()
    for d in (F32, BF):
        full = kernels.dequantize_w4(w, d)
        assert torch.equal(full.cpu().double(), q * step)                            # exactly, in either dtype


def test_weights_that_are_not_numbers():
    from rocmforge_b200 import kernels
    x = numbers(20, 128)
    x[3, 5], x[17, 100] = float("nan"), float("inf")
    w = kernels.quantize_w4(x.to(DEV), 64)
    s = unpacked(w)[1]
    nan = torch.zeros_like(s, dtype=torch.bool)
    nan[3, 0] = nan[17, 1] = True
    assert torch.equal(s.isnan(), nan)
    y = kernels.gemm_w4(kernels.quantize_q8(numbers(2, 128).to(DEV), 64), w).cpu()
    assert y[:, [3, 17]].isnan().all() and not y[:, [i for i in range(20) if i not in (3, 17)]].isnan().any()


# ---------------------------------------------------------------- products
def product_case(kind, M, N, K, G):
    from rocmforge_b200 import kernels
    w, full = weight(N, K, G)
    x = numbers(M, K, dt=BF if kind != "f32" else F32)
    if kind == "q8":
        rows = kernels.quantize_q8(x.to(DEV), G)
        return rows, stands_for(rows), w, full
    return x.to(DEV), x.double(), w, full


def terms_of(kind, K):
    """8-bit rows: an exact sum a group at least every 32, two roundings a factor.  16-bit ones: every product of a tensor-core sum may
    be cut instead of rounded, and so is every sum (2 x 2^-24 each)."""
    return K // 32 + 24 if kind == "q8" else 2 * K + 24


SIZES = [(16, 64, 32), (5, 1, 32), (33, 8, 64), (17, 100, 64), (1, 128, 128), (1003, 1100, 32), (100, 896, 128), (200, 2050, 64), (48, 19001, 128)]


@pytest.mark.parametrize("kind", ["q8", "bf16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("N,K,G", SIZES)
def test_products(kind, M, N, K, G):
    from rocmforge_b200 import kernels
    x, x64, w, full = product_case(kind, M, N, K, G)
    x64, full = x64.to(DEV), full.to(DEV)
    want, size, terms = x64 @ full.T, x64.abs() @ full.abs().T, terms_of(kind, K)
    dt = F32 if kind == "f32" else BF
    y = kernels.gemm_w4(x, w)
    assert y.dtype == dt and y.shape == (M, N)
    close(y, want, size, terms, dt)
    close(kernels.gemm_w4(x, w, out_f32=True), want, size, terms, F32)
    bias = numbers(N, seed=5)
    for b in (bias, bias.bfloat16()):
        close(kernels.gemm_w4(x, w, b.to(DEV), out_f32=True), want + b.double().to(DEV), size + b.double().abs().to(DEV), terms + 1, F32)
    h = numbers(M, N, seed=9)
    got = kernels.gemm_w4(x, w, b.to(DEV), out=h.to(DEV), accumulate=True)
    close(got, want + (h.double() + b.double()).to(DEV), size + (h.double().abs() + b.double().abs()).to(DEV), terms + 2, F32)


@pytest.mark.parametrize("M,eights,pair,ways,clusters", [(5, 1, 1, 1, 2), (8, 1, 1, 2, 1), (16, 1, 1, 2, 3), (3, 1, 1, 16, 1), (8, 1, 1, 8, 20), (15, 2, 1, 4, 2),
                                                         (16, 2, 2, 1, 1), (9, 2, 2, 4, 2), (64, 4, 1, 8, 5), (70, 4, 2, 2, 1), (1, 4, 1, 1, 1), (33, 4, 2, 1, 3), (32, 4, 2, 16, 2)])
@pytest.mark.parametrize("kind", ["q8", "bf16"])
@pytest.mark.parametrize("splits", [1, 2, 3, 8])
@pytest.mark.parametrize("N,K,G", [(300, 1088, 32), (130, 200, 64), (17, 2176, 128), (450, 77, 128)])
def test_every_way_to_share_out_a_product(monkeypatch, M, eights, pair, ways, clusters, kind, splits, N, K, G):
    """Columns over warps and over CTAs of a cluster (some of which get none), tiles over several rounds, tokens over several blocks."""
    from rocmforge_b200 import kernels
    from rocmforge_b200.kernels import quantized
    if kind == "bf16" and eights == 4:
        pytest.skip("there is no such kernel")
    monkeypatch.setattr(quantized, "w4_launch", lambda *a: (eights, pair, ways, splits, clusters))
    x, x64, w, full = product_case(kind, M, N, K, G)
    x64, full = x64.to(DEV), full.to(DEV)
    h = numbers(M, N, seed=9)
    if quantized._f("rf_gemm_w4_shared")(0 if kind == "q8" else 1, M, N, K, G, eights, pair, ways, splits, clusters) > quantized.W4_MOST_SHARED:
        with pytest.raises(kernels.KernelError, match="not supported"):
            kernels.gemm_w4(x, w, out=h.to(DEV), accumulate=True)
        return
    got = kernels.gemm_w4(x, w, out=h.to(DEV), accumulate=True)
    close(got, x64 @ full.T + h.double().to(DEV), x64.abs() @ full.abs().T + h.double().abs().to(DEV), terms_of(kind, K) + 1, F32)


@pytest.mark.parametrize("M,bn", [(1, 32), (32, 32), (40, 32), (64, 64), (33, 64), (129, 64), (128, 128), (100, 128), (300, 128), (256, 128), (20, 128)])
@pytest.mark.parametrize("splits", [1, 2, 3, 8])
@pytest.mark.parametrize("N,K,G", [(300, 1088, 32), (130, 200, 64), (17, 2176, 128), (450, 72, 128), (128, 3328, 32), (20, 8200, 128)])
def test_every_tile_on_the_tensor_cores(monkeypatch, M, bn, splits, N, K, G):
    """Tiles of tokens that are not full, rows of weights that end inside a tile, shares of the columns that are empty."""
    from rocmforge_b200 import kernels
    from rocmforge_b200.kernels import quantized
    monkeypatch.setattr(quantized, "w4_launch", lambda *a: (bn, splits))
    x, x64, w, full = product_case("bf16", M, N, K, G)
    x64, full = x64.to(DEV), full.to(DEV)
    b, h = numbers(N, seed=2), numbers(M, N, seed=9)
    got = kernels.gemm_w4(x, w, b.to(DEV), out=h.to(DEV), accumulate=True)
    close(got, x64 @ full.T + (h.double() + b.double()).to(DEV), x64.abs() @ full.abs().T + (h.double().abs() + b.double().abs()).to(DEV), terms_of("bf16", K) + 2, F32)
    close(kernels.gemm_w4(x, w), x64 @ full.T, x64.abs() @ full.abs().T, terms_of("bf16", K), BF)
    kernels.tensor_core.check_status(torch.device(DEV))


@pytest.mark.parametrize("M,K", [(513, 256), (600, 2104), (1025, 2104), (2049, 2103), (2049, 4200), (1030, 4200), (5000, 72)])
def test_many_tokens(M, K):
    """Where the weights are written out in 16 bits for the 16-bit product, in pieces of the columns for 32-bit results, and next to it."""
    from rocmforge_b200 import kernels
    x, x64, w, full = product_case("bf16", M, 130, K, 128)
    x64, full = x64.to(DEV), full.to(DEV)
    want, size, b, h = x64 @ full.T, x64.abs() @ full.abs().T, numbers(130, seed=2), numbers(M, 130, seed=9)
    close(kernels.gemm_w4(x, w), want, size, terms_of("bf16", K), BF)
    close(kernels.gemm_w4(x, w, b.to(DEV), out_f32=True), want + b.double().to(DEV), size + b.double().abs().to(DEV), terms_of("bf16", K) + 1, F32)
    close(kernels.gemm_w4(x, w, out=h.to(DEV), accumulate=True), want + h.double().to(DEV), size + h.double().abs().to(DEV), terms_of("bf16", K) + 2, F32)


@pytest.mark.parametrize("kind", ["q8", "bf16"])
def test_long_sums_are_rounded_not_cut(kind):
    """Sums of numbers of one sign, where what the tensor cores cut would add up: 40 tokens, 18,944 columns, against a 32-bit sum's error."""
    from rocmforge_b200 import kernels
    w = kernels.quantize_w4(numbers(64, 18944, spread=False).abs().to(DEV), 64)
    x = numbers(40, 18944, dt=BF, spread=False).abs().to(DEV)
    r = kernels.quantize_q8(x, 64) if kind == "q8" else x
    x64 = stands_for(r).to(DEV) if kind == "q8" else x.double()
    want = x64 @ kernels.dequantize_w4(w, F32).double().T
    # pieces of 2,048 columns: 128 additions of 16 products, each cut by at most 2^-23 of a sum that grows evenly (half of it on average); ten
    # roundings between pieces.  8-bit rows: 296 groups' roundings, two a factor
    bound = (128 / 2 + 10) * 2.0 ** -23 if kind == "bf16" else (296 / 2 + 4) * 2.0 ** -24
    err = ((kernels.gemm_w4(r, w, out_f32=True).double() - want).abs() / want).max().item()
    assert err <= bound, (err, bound)


def test_products_on_two_streams_at_once():
    """Products of every kind, clusters among them, on two streams at the same time: what they are alone."""
    from rocmforge_b200 import kernels
    w, _ = weight(1000, 8200, 128)
    xs = [numbers(M, 8200, seed=M, dt=BF).to(DEV) for M in (1, 16, 40, 300)]
    calls = [lambda x=x: kernels.gemm_w4(x, w, out_f32=True) for x in xs] + [lambda x=x: kernels.gemm_w4(kernels.quantize_q8(x, 128), w, out_f32=True) for x in xs[:3]]
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for i in range(len(calls)):
        for j, side in enumerate(streams):
            with torch.cuda.stream(side):
                got[j].append(calls[i if j == 0 else len(calls) - 1 - i]())
    torch.cuda.synchronize()
    for i, want in enumerate(alone):
        assert torch.equal(got[0][i], want) and torch.equal(got[1][len(calls) - 1 - i], want)
    kernels.tensor_core.check_status(torch.device(DEV))


@pytest.mark.parametrize("kind", ["q8", "bf16"])
def test_a_row_does_not_depend_on_its_neighbours(kind):
    from rocmforge_b200 import kernels
    w, _ = weight(96, 700, 64)
    x = numbers(8, 700, dt=BF).to(DEV)
    rows = lambda t: kernels.quantize_q8(t, 64) if kind == "q8" else t
    whole = kernels.gemm_w4(rows(x), w, out_f32=True)
    for m in (1, 3, 7):
        assert torch.equal(kernels.gemm_w4(rows(x[:m]), w, out_f32=True), whole[:m])
    bad = x.clone()
    bad[2] = float("nan")
    y = kernels.gemm_w4(rows(bad), w, out_f32=True)
    assert y[2].isnan().all() and torch.equal(y[[0, 1, 3, 4, 5, 6, 7]], whole[[0, 1, 3, 4, 5, 6, 7]])


def test_a_row_does_not_depend_on_its_neighbours_on_the_tensor_cores(monkeypatch):
    """... as long as the product is shared out in the same way, which goes by how many rows there are."""
    from rocmforge_b200 import kernels
    from rocmforge_b200.kernels import quantized
    monkeypatch.setattr(quantized, "w4_launch", lambda *a: (128, 3))
    w, _ = weight(300, 5000, 64)
    x = numbers(120, 5000, dt=BF).to(DEV)
    whole = kernels.gemm_w4(x, w, out_f32=True)
    assert torch.equal(kernels.gemm_w4(x[:110], w, out_f32=True), whole[:110])
    x[2], x[50, 4999], x[119, 0] = float("nan"), float("inf"), -float("inf")
    y = kernels.gemm_w4(x, w, out_f32=True)
    bad = [2, 50, 119]
    rest = [i for i in range(120) if i not in bad]
    assert torch.equal(y[rest], whole[rest]) and not y[bad].isfinite().any()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_16_bit_rows_any_distance_apart(M):
    from rocmforge_b200 import kernels
    w, full = weight(64, 256, 64)
    wide = numbers(M, 600, dt=BF).to(DEV)
    for c in (0, 3, 8, 344):
        x = wide[:, c:c + 256]
        close(kernels.gemm_w4(x, w, out_f32=True), x.double() @ full.to(DEV).T, x.double().abs() @ full.abs().to(DEV).T, terms_of("bf16", 256), F32)
    same = wide[:1, 8:264].expand(M, 256)                # every row the same memory
    close(kernels.gemm_w4(same, w, out_f32=True), same.double() @ full.to(DEV).T, same.double().abs() @ full.abs().to(DEV).T, terms_of("bf16", 256), F32)


def test_empty_and_refused():
    from rocmforge_b200 import kernels
    from rocmforge_b200.kernels import KernelError
    w, _ = weight(32, 128, 64)
    x = torch.zeros(3, 128, device=DEV, dtype=BF)
    r = kernels.quantize_q8(x, 64)
    assert kernels.gemm_w4(x[:0], w).shape == (0, 32)
    out = torch.zeros(3, 32, device=DEV)
    for call in (lambda: kernels.gemm_w4(x[:, :64], w), lambda: kernels.gemm_w4(kernels.quantize_q8(x, 32), w), lambda: kernels.gemm_w4(x.half(), w),
                 lambda: kernels.gemm_w4(x.t(), w), lambda: kernels.gemm_w4(x, x), lambda: kernels.gemm_w4(None, w),
                 lambda: kernels.gemm_w4(r, w, accumulate=True), lambda: kernels.gemm_w4(r, w, out=out), lambda: kernels.gemm_w4(r, w, out=out[:2], out_f32=True),
                 lambda: kernels.gemm_w4(r, w, out=torch.zeros(32, 3, device=DEV).t(), out_f32=True), lambda: kernels.gemm_w4(r, w, torch.zeros(31, device=DEV)),
                 lambda: kernels.gemm_w4(r, w, torch.zeros(32, device=DEV, dtype=torch.float16)), lambda: kernels.gemm_w4(r, w, torch.zeros(32)),
                 lambda: kernels.quantize_q8(x.t(), 64), lambda: kernels.quantize_q8(x, 16), lambda: kernels.quantize_q8(x.int(), 64),
                 lambda: kernels.quantize_w4(x.t(), 64), lambda: kernels.quantize_w4(x[:0], 64), lambda: kernels.quantize_w4(x, 256),
                 lambda: kernels.swiglu_q8(x[:, :127], 64), lambda: kernels.swiglu_q8(x, 64, activation="tanh"),
                 lambda: kernels.add_rmsnorm_q8(x, x[0], 1e-6, BF, 64), lambda: kernels.add_rmsnorm_q8(x.float(), x[0, :64], 1e-6, BF, 64),
                 lambda: kernels.add_rmsnorm_q8(x.float(), x[0], 1e-6, BF, 64, pending=x[:2]),
                 lambda: kernels.add_rmsnorm_q8(x.float(), x[0], 1e-6, BF, 64, rows=torch.zeros(2, device=DEV)),
                 lambda: kernels.add_rmsnorm_q8(torch.zeros(1, 40000, device=DEV), torch.zeros(40000, device=DEV), 1e-6, BF, 64)):
        with pytest.raises(KernelError):
            call()
    assert not out.any()


# ---------------------------------------------------------------- norm and gated unit
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,H", [(1, 64), (1, 896), (2, 100), (3, 1003), (64, 5120), (5, 8192), (1, 16384), (2, 30000), (300, 256), (300, 1600), (297, 1601)])
@pytest.mark.parametrize("pending", [None, 1, 5, 17, "same", "f32"])
def test_norm_to_8_bits(G, T, H, pending):
    from rocmforge_b200 import kernels
    h = numbers(T, H)
    w = (1 + 0.3 * numbers(H, seed=3, spread=False)).to(BF if G == 64 else F32)
    p = None
    if pending == "same":
        p = numbers(T, H, seed=4, dt=BF)
    elif pending == "f32":
        p = numbers(T, H, seed=4)
    elif pending:
        p = 0.3 * numbers(pending, T, H, seed=4)
    new = h.clone()                                       # the stream's own sum: one addend after the other, in 32 bits
    for part in ([] if p is None else p if p.dim() == 3 else [p.float()]):
        new += part
    on = h.to(DEV)
    r = kernels.add_rmsnorm_q8(on, w.to(DEV), 1e-6, BF, G, pending=None if p is None else p.to(DEV))
    assert torch.equal(on.cpu(), new)
    x = new.double()
    want = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    # the sum of squares: every square and every sum of a tree rounds, at most 45 a path; rsqrt 2 ulp; three products
    check_rows(r, want, 60 * 2.0 ** -24)
    assert r.dtype == BF and r.shape == (T, H)
    if T > 2:
        rows = torch.tensor([T - 1, 0, 0], dtype=torch.int32)
        before = on.clone()
        check_rows(kernels.add_rmsnorm_q8(on, w.to(DEV), 1e-6, BF, G, rows=rows.to(DEV)), want[rows.long()], 60 * 2.0 ** -24)
        kernels.add_rmsnorm_q8(on, w.to(DEV), 1e-6, BF, G, rows=rows.to(DEV), pending=None if p is None else p.to(DEV))
        assert torch.equal(on, before)


def test_norm_of_rows_of_zeros_and_of_no_rows():
    from rocmforge_b200 import kernels
    r = kernels.add_rmsnorm_q8(torch.zeros(2, 256, device=DEV), torch.ones(256, device=DEV), 1e-6, BF, 64)
    assert not r.q.any() and not r.scales.any()
    assert kernels.add_rmsnorm_q8(torch.zeros(0, 256, device=DEV), torch.ones(256, device=DEV), 1e-6, BF, 64).shape == (0, 256)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh"])
@pytest.mark.parametrize("T,I", [(1, 1), (1, 64), (3, 101), (2, 1030), (9, 4864), (130, 200)])
def test_gated_unit_to_8_bits(dt, G, act, T, I):
    from rocmforge_b200 import kernels
    gu = 2 * numbers(T, 2 * I, dt=dt, spread=False)
    x, u = gu.double()[:, ::2], gu.double()[:, 1::2]
    a = dict(silu=lambda: x * torch.sigmoid(x), relu=lambda: x.clamp_min(0),
             gelu_tanh=lambda: 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3))))[act]()
    r = kernels.swiglu_q8(gu.to(DEV), G, activation=act)
    full = torch.zeros(T, r.q.shape[1], dtype=torch.float64)
    full[:, :I] = a * u
    s = r.scales.cpu().double().repeat_interleave(G, 1)
    # 1 + tanh loses what tanh's last bits hold: up to 2^-22 of |x u| whatever is left; the rest is relative
    slack = (2.0 ** -22 * (x * u).abs() + 2.0 ** -20 * (a * u).abs())
    off = (r.q.cpu().double() * s - full)[:, :I].abs()
    top = full.view(T, -1, G).abs().amax(-1)
    worst = torch.zeros_like(full)
    worst[:, :I] = slack
    worst = worst.view(T, -1, G).amax(-1)
    assert ((r.scales.cpu().double() - top / 127).abs() <= worst / 127 + 2.0 ** -23 * top / 127).all()
    assert (off <= s[:, :I] * 0.5 + slack + worst.repeat_interleave(G, 1)[:, :I] + 2.0 ** -14 * s[:, :I]).all()
    assert not r.q[:, I:].any()


# ---------------------------------------------------------------- together
def test_a_layers_run_captured_and_replayed_on_another_stream():
    """norm -> product -> gated unit -> product into the stream: against the same run in 64 bits by the 8-bit rows it made itself, from a
    graph captured on a stream of its own, replayed with other numbers; the weights are made right before they are read."""
    from rocmforge_b200 import kernels
    T, H, I, G = 5, 384, 640, 64
    up, down = numbers(2 * I, H) / H ** 0.5, numbers(H, I) / I ** 0.5
    nw = torch.ones(H, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1, w2 = kernels.quantize_w4(up.to(DEV), G), kernels.quantize_w4(down.to(DEV), G)
        h, keep = torch.zeros(T, H, device=DEV), {}

        def body():
            y = kernels.add_rmsnorm_q8(h, nw, 1e-6, BF, G)
            gu = kernels.gemm_w4(y, w1)
            a = kernels.swiglu_q8(gu, G)
            kernels.gemm_w4(a, w2, out=h, accumulate=True)
            keep.update(y=y, gu=gu, a=a)
        body()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            body()
        for seed in (1, 2):
            start = numbers(T, H, seed=seed)
            h.copy_(start)
            graph.replay()
            torch.cuda.synchronize()
            f1, f2 = (kernels.dequantize_w4(w, F32).double() for w in (w1, w2))
            x = start.double()
            check_rows(keep["y"], x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt(), 60 * 2.0 ** -24)
            y64, a64 = stands_for(keep["y"]).to(DEV), stands_for(keep["a"]).to(DEV)
            close(keep["gu"], y64 @ f1.T, y64.abs() @ f1.abs().T, terms_of("q8", H), BF)
            gu = keep["gu"].cpu().double()
            check_rows(keep["a"], gu[:, ::2] * torch.sigmoid(gu[:, ::2]) * gu[:, 1::2], 2.0 ** -20)
            close(h, start.double().to(DEV) + a64 @ f2.T, start.double().abs().to(DEV) + a64.abs() @ f2.abs().T, terms_of("q8", I) + 1, F32)
    torch.cuda.current_stream().wait_stream(side)


def test_a_prompts_products_captured_and_replayed():
    """16-bit rows on the tensor cores' kernel, aligned and not, and through the weights in 16 bits, in one graph, replayed with other rows."""
    from rocmforge_b200 import kernels
    w, full = weight(200, 264, 64)
    full = full.to(DEV)
    x = torch.zeros(700, 264, device=DEV, dtype=BF)
    odd, _ = weight(48, 263, 64)
    body = lambda: (kernels.gemm_w4(x[:40], w), kernels.gemm_w4(x[:33, :263], odd), kernels.gemm_w4(x, w))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = body()
        for seed in (1, 2):
            x.copy_(numbers(700, 264, seed=seed, dt=BF))
            graph.replay()
            torch.cuda.synchronize()
            x64 = x.double()
            close(out[0], x64[:40] @ full.T, x64[:40].abs() @ full.abs().T, terms_of("bf16", 264), BF)
            close(out[2], x64 @ full.T, x64.abs() @ full.abs().T, terms_of("bf16", 264), BF)
            for now, then in zip(out, body()):
                assert torch.equal(now, then)
    torch.cuda.current_stream().wait_stream(side)


def test_tensors_of_another_device_are_refused():
    from rocmforge_b200 import kernels
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    with pytest.raises(kernels.KernelError, match="current device"):
        kernels.quantize_q8(torch.zeros(1, 64, device="cuda:1"), 64)
