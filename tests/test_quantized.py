"""Weights in 4 bits and rows in 8 bits, as far as it goes without a GPU: the stored forms and the refusals."""
import pytest
import torch

from rocmforge_b200 import kernels
from rocmforge_b200.kernels import KernelError
from rocmforge_b200.kernels.quantized import padded_columns


def unpacked(w):
    """The whole numbers and the scales of a W4Weight by the documented places, padding and all."""
    tiles, blocks = w.packed.shape[:2]
    q = torch.zeros(16 * tiles, 64 * blocks, dtype=torch.int64)
    n, k = torch.meshgrid(torch.arange(16 * tiles), torch.arange(64 * blocks), indexing="ij")
    g, r, t, c, b = n % 8, n % 16 // 8, k % 32 // 8, k % 64 // 32, k % 4
    byte = w.packed.cpu().long()[n // 16, k // 64, 4 * g + t, 8 * r + 4 * c + b]
    q = torch.where(k % 8 // 4 == 1, byte >> 4, byte & 15)
    q = torch.where(q > 7, q - 16, q)
    rows = torch.arange(16 * tiles)
    return q, w.scales.cpu()[rows // 16, :, 2 * (rows % 8) + rows % 16 // 8]


@pytest.mark.parametrize("N,K,G", [(16, 64, 32), (1, 1, 128), (17, 65, 64), (40, 130, 32), (33, 300, 128)])
def test_layout_of_weights_quantised_elsewhere(N, K, G):
    g = torch.Generator().manual_seed(N * K)
    q = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
    s = torch.rand(N, (K + G - 1) // G, generator=g).bfloat16()
    w = kernels.W4Weight.from_quantized(q, s, G)
    assert w.shape == (N, K) and w.packed.shape == ((N + 15) // 16, padded_columns(K, G) // 64, 32, 16)
    got, scales = unpacked(w)
    assert torch.equal(got[:N, :K], q.long()) and not got[N:].any() and not got[:, K:].any()
    assert torch.equal(scales[:N, :s.shape[1]], s) and not scales[N:].any() and not scales[:, s.shape[1]:].any()
    assert w.nbytes == w.packed.numel() + 2 * w.scales.numel()


def test_padded_columns():
    assert [padded_columns(k, 32) for k in (1, 64, 65)] == [64, 64, 128]
    assert [padded_columns(k, 128) for k in (1, 64, 128, 129)] == [128, 128, 128, 256]


def test_stored_forms_are_checked():
    ok = dict(packed=torch.zeros(2, 2, 32, 16, dtype=torch.uint8), scales=torch.zeros(2, 1, 16, dtype=torch.bfloat16), N=17, K=70, group=128)
    kernels.W4Weight(**ok)
    for bad in (dict(N=0), dict(K=0), dict(K=129), dict(N=33), dict(group=64), dict(group=16), dict(group=0),
                dict(packed=ok["packed"].int()), dict(packed=ok["packed"][:1]), dict(packed=ok["packed"].transpose(0, 1)),
                dict(scales=ok["scales"].float()), dict(scales=ok["scales"][:, :, :8])):
        with pytest.raises(KernelError):
            kernels.W4Weight(**{**ok, **bad})
    rows = dict(q=torch.zeros(3, 128, dtype=torch.int8), scales=torch.zeros(3, 2), K=100, group=64, dtype=torch.bfloat16)
    assert kernels.Q8Rows(**rows).shape == (3, 100)
    for bad in (dict(K=129), dict(K=64), dict(group=32), dict(group=48), dict(dtype=torch.float16), dict(q=rows["q"].to(torch.uint8)),
                dict(q=rows["q"].t().contiguous().t()), dict(scales=rows["scales"].double()), dict(scales=rows["scales"][:2])):
        with pytest.raises(KernelError):
            kernels.Q8Rows(**{**rows, **bad})


def test_what_is_not_whole_or_too_large_is_no_4_bit_weight():
    with pytest.raises(KernelError):
        kernels.W4Weight.from_quantized(torch.full((2, 64), 8), torch.ones(2, 1), 64)
    with pytest.raises(KernelError):
        kernels.W4Weight.from_quantized(torch.zeros(2, 64), torch.ones(2, 1), 64)
    with pytest.raises(KernelError):
        kernels.W4Weight.from_quantized(torch.zeros(2, 64, dtype=torch.int8), torch.ones(2, 2), 64)
    with pytest.raises(KernelError):
        kernels.W4Weight.from_quantized(torch.zeros(0, 64, dtype=torch.int8), torch.ones(0, 1), 64)


def test_nothing_runs_on_the_cpu():
    x = torch.zeros(2, 64)
    w = kernels.W4Weight.from_quantized(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 1), 64)
    r = kernels.Q8Rows(torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 1), 64, 64, torch.float32)
    for call in (lambda: kernels.quantize_w4(x), lambda: kernels.dequantize_w4(w), lambda: kernels.quantize_q8(x, 64), r.materialize,
                 lambda: kernels.add_rmsnorm_q8(x, torch.ones(64), 1e-6, torch.float32, 64), lambda: kernels.swiglu_q8(x, 32),
                 lambda: kernels.gemm_w4(r, w), lambda: kernels.gemm_w4(x, w)):
        with pytest.raises(KernelError, match="CUDA device"):
            call()


def test_options():
    from rocmforge_b200 import Options
    from rocmforge_b200.cli import build_parser
    o = Options()
    assert (o.weight_bits, o.weight_group, o.row_bits) == (16, 128, 8)
    for bad in (dict(weight_bits=8), dict(weight_bits=4, weight_group=16), dict(row_bits=4)):
        with pytest.raises(ValueError):
            Options(**bad)
    a = build_parser().parse_args(["-m", "x", "-p", "hi"])
    assert (a.weight_bits, a.weight_group, a.row_bits) == (16, 128, 8)


def test_products_of_a_part():
    """Which products a model's parts offer for 4 bits: the projections of attention and of dense feed-forwards."""
    from helpers import CONFIGS, config_dict
    from rocmforge_b200.config import Qwen2Config, architecture_for
    from rocmforge_b200.parts.attention import GQAAttention
    from rocmforge_b200.parts.mlp import GatedMLP
    cfg = Qwen2Config.from_dict(config_dict(CONFIGS["A"]))
    spec = architecture_for(cfg.architecture).build(cfg)
    offering = {type(p) for p in spec.named_parts().values() if type(p).linears is not __import__("rocmforge_b200.parts.base", fromlist=["Part"]).Part.linears}
    assert offering == {GQAAttention, GatedMLP}


B200_CLUSTERS = (148, 74, 45, 33, 26, 22, 15, 15)         # of 1 .. 8 blocks that run at once


def clusters(splits):
    return B200_CLUSTERS[splits - 1]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (1003, 1100), (896, 896), (4608, 3584), (37888, 3584), (3584, 18944), (152064, 8192), (64, 70000)])
def test_how_products_are_shared_out(q8, N, K):
    """Every plan fits into shared memory, has a kernel, and its clusters run at once; no block of a cluster is left without a stage."""
    from rocmforge_b200.kernels import quantized
    for group in (32, 64, 128):
        for M in (1, 8, 9, 16, 17, 32, 33, 64, 100, 128, 129, 200, 2000, 100000):
            plan = quantized.w4_launch(q8, M, N, K, group, clusters)
            if plan is None:
                assert q8 and K == 70000 and M > 8
            elif len(plan) == 2:
                bn, splits = plan
                assert not q8 and (M > 8 or K == 70000) and bn in (32, 64, 128) and 1 <= splits <= min(8, (K + 511) // 512)
            else:
                eights, pair, ways, splits, used = plan
                assert (q8, eights, pair) in quantized.W4_COST and ways in (1, 2, 4, 8, 16) and 1 <= splits <= 8 and (q8 or M <= 128)
                assert quantized._f("rf_gemm_w4_shared")(0 if q8 else 1, M, N, K, group, *plan) <= quantized.W4_MOST_SHARED
                assert used >= 1 and (used == 1 or used * ((M + 8 * eights - 1) // (8 * eights)) <= clusters(splits))
                assert eights * 8 >= min(M, 16) or K > 18944
    assert quantized.w4_launch(False, 16, 37888, 3584, 128, clusters) == (2, 1, 1, 1, 148)
    assert quantized.w4_launch(False, 32, 37888, 3584, 128, clusters) == (32, 1)
    assert quantized.w4_launch(False, 64, 3584, 18944, 128, clusters) == (64, 4)
