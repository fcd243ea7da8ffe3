"""Edges of the 4-bit weight path that show without a GPU: what the sources say, and what the host decides."""
import pytest
import torch

from test_wait_rules import kernels as sources


def body_of(name):
    return next(body for n, _, body in sources() if n == name)


def test_chosen_rows_are_read_after_the_wait():
    """``add_rmsnorm_q8(rows=...)`` takes indices from anywhere, the kernel launched just before it among them."""
    body = body_of("add_rmsnorm_q8_kernel")
    assert body.index("pdl_wait(pending, rows)") < body.index("rows[")


B200_CLUSTERS = (148, 74, 45, 33, 26, 22, 15, 15)         # of 1 .. 8 blocks that run at once


def clusters(splits):
    return B200_CLUSTERS[splits - 1]


@pytest.mark.parametrize("M", [1, 17, 64, 129, 700, 5000])
@pytest.mark.parametrize("N,K", [(16, 64), (37888, 3584), (3584, 18944), (64, 200000)])
def test_plans_without_the_tcgen05_kernels(M, N, K):
    from rocmforge_b200.kernels import quantized
    plan = quantized.w4_launch(False, M, N, K, 64, clusters, False)
    assert (plan is None) == (K == 200000) or len(plan) == 5
    if plan is not None:
        assert quantized._f("rf_gemm_w4_shared")(1, M, N, K, 64, *plan) <= quantized.W4_MOST_SHARED and (False, *plan[:2]) in quantized.W4_COST


@pytest.mark.parametrize("group", [32, 64, 128])
def test_long_8_bit_rows_go_a_few_at_a_time(group):
    """Rows that do not lie in shared memory together have a plan for fewer of them: as many as fit."""
    from rocmforge_b200.kernels import quantized
    whole = 0
    for K in (18944, 70000, 100000, 140000, 300000, 400000):
        for M in (1, 2, 8, 9, 32, 100):
            step = quantized.q8_rows_at_once(M, 64, K, group, clusters)
            assert step is not None and 1 <= step <= M and quantized.w4_launch(True, step, 64, K, group, clusters)
            whole += step < M
            assert step == M or quantized.w4_launch(True, M, 64, K, group, clusters) is None
    assert whole > 0 and quantized.q8_rows_at_once(1, 64, 4000000, group, clusters) is None


@pytest.mark.parametrize("name,parts", [("RA", {"GQAAttention", "SquaredReluMLP"}), ("RB", {"GQAAttention", "SquaredReluMLP"}), ("FA", {"GQAAttention", "GatedMLP"}),
                                        ("VA", {"GQAAttention"}), ("GA", {"GatedMLP"}), ("DC", {"GQAAttention", "GatedMLP"})])
def test_products_of_every_kind_of_part(folders, name, parts):
    """Which products the parts of other designs offer for 4 bits, bound: all that their matrices go into, the one that alone reads the input first."""
    from rocmforge_b200.config import load_config
    from rocmforge_b200.weights import load_folder
    folder = folders(name, "bfloat16")
    arch, config = load_config(folder)
    spec = arch.build(config)
    params, offering = load_folder(folder, spec.param_specs(), torch.bfloat16, "cpu"), set()
    for prefix, part in spec.named_parts().items():
        specs = part.param_specs()
        if type(part).__name__ not in parts:
            continue
        part.bind({k[len(prefix):]: t for k, t in params.items() if k.startswith(prefix) and k[len(prefix):] in specs}, torch.bfloat16)
        offering.add(type(part).__name__)
        linears = part.linears()
        matrices = [s for s in specs.values() if s.kind == "matrix"]
        assert len(linears) == 2 and part.input_weight() is linears[0].weight
        assert sum(a.weight.numel() for a in linears) >= sum(s.shape[0] * s.shape[1] for s in matrices) and linears[0].K == part.hidden == linears[1].N
    assert offering == parts
