"""A model whose keys and values are held in 4 bits, against the plain model over rows that are quantised as the format says, and
steps with shared pages and recorded launches against each request alone."""

import pytest
import torch

import helpers
import plain_packed
import plain_qwen2
from helpers import TINY_A, TINY_B, TINY_D

pytestmark = pytest.mark.gpu
DEV = "cuda"
WHOLE_D = dict(TINY_D, use_sliding_window=False)  # every layer keeps all keys: pages can be shared
CONFIGS = {"head-32": dict(TINY_A, head_dim=32), "window-21": TINY_B, "head-64": WHOLE_D, "head-64-window-48": TINY_D}


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    from ferrisinfer_b200.kernels import ops

    ops.require_device()
    yield
    torch.cuda.synchronize()
    ops.check_kernel_status()


def runner_of(folder, dtype, **more):
    from ferrisinfer_b200.engine.runner import ModelRunner
    from ferrisinfer_b200.weights import load_model

    model, _ = load_model(folder, dtype, DEV, cache_bits=4)
    return ModelRunner(model, dtype, torch.device(DEV), page_size=16, num_pages=200, max_requests=8, **more)


def quantised(x):
    """What rows [n, kv heads, D] stand for once they are in the cache."""
    s = plain_packed.scales_of(x).double()
    scale, least = (s[..., i].repeat_interleave(32, -1) for i in range(2))
    code = ((x.double() - least) / scale).round().clamp(0, 15)
    return (torch.where(scale > 0, code, torch.zeros_like(code)) * scale + least).to(x.dtype)


@pytest.mark.parametrize("layers", [1, 2])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_32_bit_logits_are_the_plain_models_over_quantised_rows(tmp_path, monkeypatch, name, layers):
    config = dict(CONFIGS[name], num_hidden_layers=layers, max_window_layers=layers - 1)
    folder = helpers.make_folder(tmp_path, config, seed=4, score_std=1.0)
    _, weights = helpers.read_folder(folder)
    ids = {f"r{i}": helpers.random_ids(config["vocab_size"], n, 60 + i) for i, n in enumerate((70, 33, 9, 100))}
    whole = helpers.oracle_logits(config, weights, ids)
    plain_attention = plain_qwen2.attention
    monkeypatch.setattr(plain_qwen2, "attention", lambda q, k, v, *rest: plain_attention(q, quantised(k), quantised(v), *rest))
    want = helpers.oracle_logits(config, weights, ids)
    apart = lambda a, b: sum(float((a[at] - b[at]).double().norm()) ** 2 for at in want) ** 0.5
    four_bits = apart(whole, want)
    assert four_bits > 0.005 * sum(float(row.double().norm()) ** 2 for row in want.values()) ** 0.5
    for trace in (helpers.trace_whole(ids), helpers.trace_portions(ids), helpers.trace_tail_decoded(ids, 12), helpers.trace_mixed(ids, 3)):
        got = helpers.replay(runner_of(folder, torch.float32), trace)
        # 32-bit projections move a code by one where its quotient lies beside a tie, about one in ten thousand, an error of one step
        # where rounding to codes leaves 0.29 of a step everywhere: 0.035 of what the four bits cost; a second layer's rows then
        # differ a little everywhere, and several in a thousand of its codes with them.
        assert apart(got, want) < (0.1 if layers == 1 else 0.4) * four_bits


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_shared_pages_and_recorded_steps_give_what_each_request_gets_alone(tmp_path, dtype):
    """Requests with the same beginning, decoded together from recorded steps: every token is (within what steps of another size
    may move a logit) the greatest of the request's logits from one whole prompt, without recording or sharing."""
    from ferrisinfer_b200 import Engine, SamplingParams, SchedulerConfig
    from ferrisinfer_b200.engine.runner import StepEntry

    folder, vocab = helpers.make_folder(tmp_path, WHOLE_D, seed=5, score_std=1.0), WHOLE_D["vocab_size"]
    base = helpers.random_ids(vocab, 50, 1)
    asked = [base, base[:48] + helpers.random_ids(vocab, 7, 2), base[:33] + helpers.random_ids(vocab, 40, 3), helpers.random_ids(vocab, 33, 4)]
    params = SamplingParams.greedy(max_new_tokens=14)
    engine = Engine(folder, dtype=dtype, num_pages=200, cache_bits=4,
                    scheduler=SchedulerConfig(max_batch_size=8, max_prefill_chunk_tokens=32, max_sequence_length=256, min_prefix_share_tokens=16))
    numbers = [engine.submit(asked[0], params)]
    while not engine.scheduler.running or engine.scheduler.running[0].num_computed < len(base):
        engine.step()  # until the first prompt is in the cache
    numbers += [engine.submit(p, params) for p in asked[1:]]
    while engine.has_unfinished():
        engine.step()
    outs = [engine.output_of(n) for n in numbers]
    assert engine.runner.graph_replays > 5 and engine.runner.cache.stats["shared_tokens"] == 48 + 32
    torch_dtype = torch.bfloat16 if dtype == "bfloat16" else torch.float32
    for prompt, out in zip(asked, outs):
        tokens = out.generated_token_ids()
        assert len(tokens) == 14
        runner = runner_of(folder, torch_dtype, cuda_graphs=False, prefix_sharing=False)
        ids = prompt + tokens[:-1]
        rows = runner.step([StepEntry("r", ids, list(range(len(prompt) - 1, len(ids))))]).clone()
        assert runner.graph_replays == 0
        # the bound that whole prompts and portions of them keep to, for the token's logit and for the greatest
        slack = 2 * rows.abs().max() * (0.05 if dtype == "bfloat16" else 0.01)
        picked = rows.gather(1, torch.tensor(tokens, device=DEV)[:, None])[:, 0]
        assert (picked >= rows.max(1).values - slack).all(), (rows.max(1).values - picked, slack)
        assert slack < 0.7 * (rows.max(1).values - rows.mean(1)).min()  # (a token at random would not do)
