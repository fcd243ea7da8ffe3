"""Models with 4-bit weights through the engine: every design against itself with the same weights held in 16 (32) bits."""
import os
import subprocess
import sys

import pytest
import torch

from helpers import BF16_REL_TO_MAX, CONFIGS, F32_ATOL, F32_RTOL, ROOT, random_tokens

pytestmark = pytest.mark.gpu
TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def pair(folders, name, dtype, group, row_bits):
    """(the model with 4-bit weights, one that holds the numbers which those stand for)"""
    import rocmforge_b200 as rf
    from rocmforge_b200 import kernels
    four = rf.Model.from_folder(folders(name, dtype), dtype=TORCH[dtype], options=rf.Options(weight_bits=4, weight_group=group, row_bits=row_bits))
    full = rf.Model.from_folder(folders(name, dtype), dtype=TORCH[dtype])
    held = 0
    for prefix, part in full.spec.named_parts().items():
        for a, b in zip(part.linears(), four.spec.named_parts()[prefix].linears()):
            assert isinstance(b.weight, kernels.W4Weight) and b.weight.group == group and b.weight.shape == a.weight.shape
            a.weight = kernels.dequantize_w4(b.weight, TORCH[dtype])
            held += a.weight.numel() * a.weight.element_size() - b.weight.nbytes
    assert held > 0 and four.weight_bytes == full.weight_bytes - held
    return four, full


def assert_both_close(a, b, dtype, what):
    """Two runs of the engine, each of which may be as far from the plain model as the engine's tests allow: twice that apart."""
    a, b = a.double(), b.double()
    bound = 2 * (F32_ATOL + F32_RTOL * b.abs() if dtype == "float32" else BF16_REL_TO_MAX * b.abs().max())
    assert torch.isfinite(a).all() and a.shape == b.shape and ((a - b).abs() <= bound).all(), f"{what}: {float((a - b).abs().max())}"


def run_both(four, full, prompts, vocab, decode=3):
    """Logits of a step of prompts and of some steps of one token, of both models."""
    import rocmforge_b200 as rf
    out = []
    for m in (four, full):
        cache = m.new_cache(max_tokens=64 * 24, max_slots=4)
        slots = [cache.alloc_slot() for _ in prompts]
        got = [m.step(cache, [rf.StepRequest(s, p, [0, len(p) - 1] if len(p) > 1 else [0]) for s, p in zip(slots, prompts)])]
        for d in range(decode):
            got.append(m.step(cache, [rf.StepRequest(s, [random_tokens(vocab, 1, 10 * d + i)[0]], [0]) for i, s in enumerate(slots)]))
        out.append(torch.cat(got).cpu())
    return out


DESIGNS = ["A", "B", "C", "D", "E", "RA", "RB", "VA", "VD", "FA", "FC", "LA", "LC", "GA", "GE", "DA", "DC"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", DESIGNS)
def test_rows_as_they_are(folders, name, dtype):
    """Prompts of few and of many tokens (one step of 150, beyond what products of few tokens take), then single tokens: the same numbers
    are multiplied, so the usual bounds hold."""
    four, full = pair(folders, name, dtype, 64 if name in ("B", "RB") else 32, 16)
    V = four.spec.vocab_size
    longest = min(100, four.spec.max_position - 8)
    for lens in ((5, 17), (longest, 51)):
        a, b = run_both(four, full, [random_tokens(V, n, n) for n in lens], V)
        assert_both_close(a, b, dtype, f"{name} {dtype} {lens}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", DESIGNS)
def test_rows_in_8_bits(folders, name, dtype):
    """A number in 8 bits is off by at most half of 1/127 of its group's largest, 0.29 / 127 of it on average (rms); with the largest at 2.5
    times a group's rms that is 0.6 % of a product's input.  Every layer has four such inputs and up to four layers pass them on; added up
    without any cancellation that is 10 % of the logits' rms, of which the models here may use up a half more where a norm or a cap
    follows a sum that has cancelled."""
    four, full = pair(folders, name, dtype, 32, 8)
    V = four.spec.vocab_size
    a, b = run_both(four, full, [random_tokens(V, n, n) for n in (5, 17)], V)
    assert torch.isfinite(a).all()
    off = float((a.double() - b.double()).norm() / b.double().norm())
    assert 0 < off < 0.15, off


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("row_bits", [8, 16])
def test_replayed_steps_are_the_plain_steps(folders, dtype, row_bits):
    import rocmforge_b200 as rf
    prompts = [random_tokens(300, n, n) for n in (3, 30, 64)]
    options = dict(weight_bits=4, weight_group=64, row_bits=row_bits)
    a = rf.LLM(folders("D", dtype), dtype=dtype, options=rf.Options(decode_graphs=True, **options))
    b = rf.LLM(folders("D", dtype), dtype=dtype, options=rf.Options(decode_graphs=False, **options))
    ra = a.generate(prompts, max_tokens=70, temperature=0.0, stop_token_ids=[])
    rb = b.generate(prompts, max_tokens=70, temperature=0.0, stop_token_ids=[])
    assert a.engine.decode_runner.replays > 0 and b.engine.decode_runner is None
    assert [r.tokens for r in ra] == [r.tokens for r in rb]


def test_two_graphs_and_an_eager_step_share_nothing(folders):
    """Decode graphs of two batch sizes, replayed in turn with steps outside graphs between them: every sequence goes on as it does alone."""
    import rocmforge_b200 as rf
    options = rf.Options(weight_bits=4, weight_group=64)
    llm = rf.LLM(folders("D", "bfloat16"), options=options)
    prompts = [random_tokens(300, n, n) for n in (40, 21, 33)]
    alone = [llm.generate([p], max_tokens=12, temperature=0.0, stop_token_ids=[])[0].tokens for p in prompts]
    both = llm.generate(prompts[:2], max_tokens=12, temperature=0.0, stop_token_ids=[])
    again = [llm.generate([p], max_tokens=12, temperature=0.0, stop_token_ids=[])[0].tokens for p in prompts]
    assert again == alone and all(len(r.tokens) == 12 for r in both)


@pytest.mark.parametrize("width", [(3584, 18944, 28, 4), (896, 4864, 14, 2)])
def test_real_widths(width):
    """One layer of the 7B and the 0.5B shape, 64 and 1 tokens."""
    import rocmforge_b200 as rf
    from rocmforge_b200 import kernels
    from rocmforge_b200.config import Qwen2Config
    H, I, nh, nkv = width
    cfg = Qwen2Config.from_dict(dict(CONFIGS["D"], num_hidden_layers=1, hidden_size=H, intermediate_size=I, num_attention_heads=nh, num_key_value_heads=nkv,
                                     head_dim=H // nh))
    four = rf.Model.random(cfg, 5, options=rf.Options(weight_bits=4, row_bits=16))
    full = rf.Model.random(cfg, 5)
    for prefix, part in full.spec.named_parts().items():
        for a, b in zip(part.linears(), four.spec.named_parts()[prefix].linears()):
            a.weight = kernels.dequantize_w4(b.weight)
    for lens in ((64,), (1, 1), (200,)):
        a, b = run_both(four, full, [random_tokens(520, n, n + i) for i, n in enumerate(lens)], 520)
        assert_both_close(a, b, "bfloat16", f"{width} {lens}")


def test_command_line(folders):
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "rocmforge"), "--model", folders("A", "bfloat16"), "--prompt-ids", "1,2,3",
                          "--max-tokens", "4", "--temperature", "0", "--weight-bits", "4", "--weight-group", "32", "--row-bits", "8"],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
