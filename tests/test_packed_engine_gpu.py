"""The packed cache where it is used: an engine whose keys and values are held in 4 bits, and a cache that keeps to a budget."""

import os
import sys

import pytest
import torch

import plain_packed as plain
from helpers import TINY_A, TINY_B, TINY_D

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEAD_32 = dict(TINY_A, head_dim=32)


def engine(config, dtype, **more):
    from ferrisinfer_b200 import Engine

    return Engine(config=config, seed=3, dtype=dtype, num_pages=200, **more)


def prompts(vocab, lengths, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in lengths]


@pytest.mark.parametrize("config", [HEAD_32, TINY_B, TINY_D], ids=["head-32", "window-21", "head-64-window-48"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_steps_match_one_whole_prompt(config, dtype):
    """Portions, single tokens and a whole prompt see the same cache: the logits after the same tokens agree."""
    from ferrisinfer_b200.engine.runner import StepEntry

    ids = prompts(config["vocab_size"], [75])[0]
    got = []
    for cut in ([75], [40, 35], [1] * 10 + [50] + [1] * 15):
        e = engine(config, dtype, cache_bits=4)
        at = 0
        for n in cut:
            logits = e.runner.step([StepEntry("r", ids[at:at + n], [n - 1])])
            at += n
        got.append(logits.clone())
    scale = got[0].abs().max()
    # The codes of a token's keys and values come from the same numbers only up to the rounding of its projections, whose kernels
    # differ with the number of rows: a code may change by one, a fifteenth of its group's spread.
    for other in got[1:]:
        assert (other - got[0]).abs().max() <= scale * (0.05 if dtype == "bfloat16" else 0.01)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_four_bits_stay_near_the_whole_cache(dtype):
    from ferrisinfer_b200.engine.runner import StepEntry

    ids = prompts(TINY_D["vocab_size"], [60])[0]
    logits = [engine(TINY_D, dtype, **more).runner.step([StepEntry("r", ids, list(range(60)))]).clone() for more in ({}, {"cache_bits": 4})]
    off = (logits[0] - logits[1]).norm() / logits[0].norm()
    assert 0 < off < 0.1


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generation_with_shared_pages_and_recorded_steps(dtype):
    """Requests of all lengths, decoded from recorded steps, some with the beginning of another: the tokens that each gets alone."""
    from ferrisinfer_b200 import SamplingParams

    base = prompts(TINY_D["vocab_size"], [50])[0]
    asked = [base, base[:48] + prompts(TINY_D["vocab_size"], [7], 5)[0], base[:17], prompts(TINY_D["vocab_size"], [33], 6)[0]]
    params = SamplingParams.greedy(max_new_tokens=12)
    together = [o.generated_token_ids() for o in engine(TINY_D, dtype, cache_bits=4).generate(asked, params)]
    again = [o.generated_token_ids() for o in engine(TINY_D, dtype, cache_bits=4).generate(asked, params)]
    assert together == again and all(len(t) == 12 for t in together)


def test_pages_that_fit_and_refusals():
    from ferrisinfer_b200 import Engine
    from ferrisinfer_b200.kernels import ops

    e = engine(TINY_D, "bfloat16", cache_bits=4)
    caches = [c for c in e.runner.cache.layer_caches if c is not None]
    assert all(c.packed is not None and c.k is None and c.packed.pages == 201 for c in caches)
    assert ops.PackedPages.bytes_per_token(2, 64) == 160  # 5 bits an element
    for config, bits in ((TINY_D, 8), (TINY_A, 4)):  # other widths; heads of 16
        with pytest.raises(ValueError):
            Engine(config=config, seed=0, cache_bits=bits, num_pages=8)


@pytest.mark.parametrize("heads, kv_heads, D", [(4, 2, 64), (6, 1, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_budget_is_kept_by_weight(heads, kv_heads, D, dtype):
    """Portions and single tokens over a cache with a budget: outputs against plain attention over the rows that it says it
    kept, and rows kept against the weights that plain attention gives them."""
    from ferrisinfer_b200.cache.budget import BudgetedCache

    cache = BudgetedCache(3, kv_heads, D, budget=48, slack=10, keep_first=2, keep_last=8, max_portion=40, page_size=16)
    first, second = cache.admit(), cache.admit()
    gen = torch.Generator(device=DEV).manual_seed(2)
    held = {r: [None] * kv_heads for r in (first, second)}  # per head: keys, values, weights of the rows held, 64 bits
    evicted = 0
    for lens in ([40, 7], [30, 40], [1, 20], [1, 1], [40, 1], [1, 30], [33, 1]):
        T = sum(lens)
        qkv = torch.randn(T, (heads + 2 * kv_heads) * D, generator=gen, device=DEV).to(dtype)
        k, v = qkv[:, heads * D:(heads + kv_heads) * D], qkv[:, (heads + kv_heads) * D:]
        out = torch.empty(T, heads * D, dtype=dtype, device=DEV)
        before = {r: cache.rows(r) for r in held}
        cache.step([first, second], lens, qkv, k, v, out, heads, D ** -0.5)
        at = 0
        for r, n in ((first, lens[0]), (second, lens[1])):
            one = plain.cache_of(k[at:at + n].reshape(n, kv_heads, D), v[at:at + n].reshape(n, kv_heads, D), 16)
            new_k, new_v, _ = plain.request_rows(one, list(range(-(-n // 16))), n, 16)
            G = heads // kv_heads
            for h in range(kv_heads):
                old = held[r][h] or (new_k[:0, h], new_v[:0, h], torch.zeros(0, dtype=torch.float64, device=DEV))
                kk, vv = torch.cat([old[0], new_k[:, h]]), torch.cat([old[1], new_v[:, h]])
                q = qkv[at:at + n, h * G * D:(h + 1) * G * D].double().view(n, G, D)
                want, w, size, _ = plain.attend(q, kk[:, None], vv[:, None], torch.ones(len(kk), dtype=torch.bool, device=DEV), before[r], D ** -0.5)
                got = out[at:at + n, h * G * D:(h + 1) * G * D].double().view(n, G, D)
                # weights rounded to eleven bits, outputs to eight (bf16 rows); sums of 32 bits
                assert ((got - want).abs() <= (size + 4) * (2.0 ** -10 if dtype == torch.bfloat16 else 2.0 ** -17) + want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 0)).all()
                held[r][h] = (kk, vv, torch.cat([old[2], torch.zeros(n, dtype=torch.float64, device=DEV)]) + w[0])
            total = before[r] + n
            if total > 58:
                evicted += 1
                assert cache.rows(r) == 48
                for h in range(kv_heads):
                    kept = cache.last_kept[r][h].long()
                    kk, vv, w = held[r][h]
                    assert (kept[1:] > kept[:-1]).all() and kept[0] == 0 and kept[1] == 1 and kept[-8:].tolist() == list(range(total - 8, total))
                    out_of = torch.ones(total, dtype=torch.bool, device=DEV)
                    out_of[kept] = False
                    assert w[kept[2:-8]].min() >= w[out_of].max() * (1 - 1e-4)
                    held[r][h] = (kk[kept], vv[kept], w[kept])
            else:
                assert cache.rows(r) == total
            for h in range(kv_heads):
                w = held[r][h][2]
                assert ((cache.weights(r)[h].double() - w).abs() <= 1e-4 * w + 1e-9).all()
            at += n
    assert evicted == cache.evictions > 4
    cache.release(second)
    cache.release(first)
    assert cache.pool.num_used == 0


def test_a_budget_refuses():
    from ferrisinfer_b200.cache.budget import BudgetedCache
    from ferrisinfer_b200.errors import CacheError

    with pytest.raises(CacheError):
        BudgetedCache(1, 1, 64, budget=8, keep_first=4, keep_last=5)
    cache = BudgetedCache(1, 1, 64, budget=16, keep_last=4, max_portion=8)
    r = cache.admit()
    x = torch.zeros(9, 64, device=DEV)
    for requests, lens in (([r], [9]), ([r, r], [4, 5]), ([r + 1], [9]), ([r], [8]), ([], [])):
        with pytest.raises(CacheError):
            cache.step(requests, lens, x, x, x, x, 1, 1.0)
    with pytest.raises(CacheError):
        cache.admit()
    cache.release(r)
    with pytest.raises(CacheError):
        cache.rows(r)


def test_the_example_runs():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import endless_request

    result = endless_request.main(["--tokens", "1500", "--budget", "400", "--heads", "4", "--head-dim", "64"])
    assert result["evictions"] > 0 and max(result["rows held"]) <= 400 + 128
    assert result["bytes held"] < result["bytes of everything in bf16"] / 5


def test_a_model_folder_and_the_command_line(tmp_path, capsys):
    from ferrisinfer_b200 import Engine, SamplingParams
    from ferrisinfer_b200.cli.main import main
    from helpers import make_folder

    folder = make_folder(tmp_path / "model", TINY_D, seed=1, score_std=1.0)
    out = Engine(str(folder), dtype="bfloat16", num_pages=64, cache_bits=4).generate([[1, 2, 3, 4]], SamplingParams.greedy(max_new_tokens=5))
    assert main(["generate-hf", "1,2,3,4", "5", "--model", str(folder), "--num-pages", "64", "--cache-bits", "4"]) == 0
    assert str(out[0].generated_token_ids()[-1]) in capsys.readouterr().out
