"""Decoding by trees of drafted tokens: the operators of a step one after the other, recorded, on other streams, from two threads."""

import random
import threading

import pytest
import torch

from test_tree_gpu import DEV, Step, drafted_step, ints, nothing_reported, ops, rng, tree  # noqa: F401

pytestmark = pytest.mark.gpu
HEADS, KV_HEADS, D, PAGE, V, PAGES, BLOCKS = 4, 2, 64, 16, 97, 60, 12


class Decoder:
    """One layer of attention between an embedding and a vocabulary, 32 bits, greedy."""

    def __init__(self, ops, requests):
        from ferrisinfer_b200.engine.workspace import Workspace

        gen = rng(5)
        self.ops, self.workspace = ops, Workspace(DEV)
        self.embedding = torch.randn(V, 80, generator=gen, device=DEV)
        self.qkv = torch.randn(80, (HEADS + 2 * KV_HEADS) * D, generator=gen, device=DEV) / 8
        self.head = torch.randn(HEADS * D, V, generator=gen, device=DEV)
        self.freq = (10000.0 ** (-torch.arange(0, D, 2, device=DEV) / D)).float()
        self.k, self.v = (torch.full((PAGES, KV_HEADS, PAGE, D), float("nan"), device=DEV) for _ in range(2))
        self.layers = ops.CacheLayers([(self.k, self.v)])
        order = random.Random(2).sample(range(PAGES), PAGES)
        self.tables = [order[i * BLOCKS:(i + 1) * BLOCKS] for i in range(requests)]
        self.table = ints(self.tables)

    def places(self, request, rows):
        return [self.tables[request][r // PAGE] * PAGE + r % PAGE for r in rows]

    def rotated(self, tokens, positions, slots):
        qkv = self.embedding[tokens.long()] @ self.qkv
        self.ops.rope_cache_write(qkv, positions, self.freq, slots, self.k, self.v, HEADS, KV_HEADS, D, D, PAGE)
        return qkv

    def prompt(self, request, tokens):
        """All tokens but the last into the cache; the step that follows brings that."""
        n = len(tokens) - 1
        if n:
            self.rotated(ints(tokens[:n]), ints(list(range(n))), ints(self.places(request, range(n))))

    def step(self, x, most_nodes, most_rows):
        """A step on the device, from inputs there; everything that it leaves is in ``x``."""
        ops = self.ops
        qkv = self.rotated(x["tokens"], x["positions"], x["slots"])
        out = torch.zeros(qkv.shape[0], HEADS * D, device=DEV)
        ops.tree_attention(qkv, out, self.k, self.v, self.table, x["q_start"], x["starts"], x["parents"], most_nodes, most_rows, HEADS, D ** -0.5, workspace=self.workspace)
        x["logits"] = out @ self.head
        ops.sampling_probs(x["logits"], x["logits"])
        ops.verify_tree(x["logits"], x["tokens"], x["parents"], x["q_start"], x["uniforms"], x["nodes"], x["accepted"], x["token"])
        ops.keep_tree_rows(self.layers, self.table, x["starts"], x["nodes"], x["accepted"])


def inputs(decoder, roots, starts, trees):
    """trees: (parents, tokens) of every request, the root first."""
    x = {"tokens": [], "parents": [], "positions": [], "slots": [], "q_start": [0], "starts": starts}
    for r, (parents, tokens) in enumerate(trees):
        depth = []
        for p in parents:
            depth.append(0 if p < 0 else depth[p] + 1)
        x["tokens"] += [roots[r]] + tokens[1:]
        x["parents"] += parents
        x["positions"] += [starts[r] + d for d in depth]
        x["slots"] += decoder.places(r, range(starts[r], starts[r] + len(parents)))
        x["q_start"].append(len(x["tokens"]))
    x = {k: ints(v) for k, v in x.items()}
    S, most = len(trees), max(len(p) for p, _ in trees)
    x.update(uniforms=torch.rand(len(x["tokens"]), generator=rng(1), device=DEV), nodes=ints([[0] * most] * S), accepted=ints([0] * S), token=ints([0] * S))
    return x


PROMPTS = [[3, 14, 15], [9] + list(range(40, 70)), [26]]
STEPS = 40


@pytest.fixture(scope="module")
def token_by_token(ops):
    """What the requests go on with, each token by a step of its own."""
    decoder, texts = Decoder(ops, 3), [list(p) for p in PROMPTS]
    for r, p in enumerate(PROMPTS):
        decoder.prompt(r, p)
    for _ in range(STEPS):
        starts = [len(t) - 1 for t in texts]
        x = inputs(decoder, [t[-1] for t in texts], starts, [([-1], [0])] * 3)
        decoder.step(x, 1, max(starts) + 1)
        # (what the next token is does not hang on a rounding: the greatest logit is alone)
        assert (x["logits"].sum(-1) == 1).all() and (x["accepted"] == 0).all()
        for t, token in zip(texts, x["token"].tolist()):
            t.append(token)
    return texts


def drafted(texts, whole, rng_, nodes):
    """A tree for every request: branches of the text that is to come, with wrong tokens among them."""
    trees = []
    for t, text in zip(texts, whole):
        parents, tokens, depth, right = [-1], [t[-1]], [0], [True]
        for i in range(1, nodes):
            p = rng_.randrange(max(0, i - 4), i)
            d = depth[p] + 1
            follows = text[len(t) - 1 + d] if len(t) - 1 + d < len(text) else 0
            good = right[p] and rng_.random() < 0.7
            parents.append(p), depth.append(d), right.append(good)
            tokens.append(follows if good else (follows + 1 + rng_.randrange(V - 1)) % V)
        trees.append((parents, tokens))
    return trees


@pytest.mark.parametrize("nodes", [2, 9, 23])
@pytest.mark.parametrize("recorded", [False, True], ids=["called", "recorded"])
def test_trees_go_on_as_tokens_do(ops, token_by_token, nodes, recorded):
    decoder, texts, draw = Decoder(ops, 3), [list(p) for p in PROMPTS], random.Random(nodes)
    for r, p in enumerate(PROMPTS):
        decoder.prompt(r, p)
    graph, x, steps, most_rows = None, None, 0, BLOCKS * PAGE
    while min(len(t) - len(p) for t, p in zip(texts, PROMPTS)) < STEPS - 12:
        starts = [len(t) - 1 for t in texts]
        now = inputs(decoder, [t[-1] for t in texts], starts, drafted(texts, token_by_token, draw, nodes))
        if not recorded:
            x = now
            decoder.step(x, nodes, most_rows)
        elif graph is None:
            x = now
            k, v = decoder.k.clone(), decoder.v.clone()
            decoder.step(x, nodes, most_rows)  # (everything has its memory and its library's handles)
            decoder.k.copy_(k), decoder.v.copy_(v)
            decoder.workspace.pin()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                decoder.step(x, nodes, most_rows)
            graph.replay()
        else:
            for name in ("tokens", "parents", "positions", "slots", "q_start", "starts", "uniforms"):
                x[name].copy_(now[name])
            graph.replay()
        ops.check_kernel_status()
        for r, t in enumerate(texts):
            path = x["nodes"][r].tolist()
            tokens = x["tokens"].tolist()[r * nodes:(r + 1) * nodes]
            n = int(x["accepted"][r])
            assert path[0] == 0 and all(i == -1 for i in path[n + 1:])
            t += [tokens[i] for i in path[1:n + 1]] + [int(x["token"][r])]
            del t[len(token_by_token[r]):]  # (beyond what is known)
            assert t == token_by_token[r][:len(t)]
        steps += 1
    assert steps < (STEPS - 12 if nodes > 2 else STEPS)  # (some of what was drafted was taken)


def last_steps():
    """Inputs for each of the operators behind the attention, and what they leave."""
    gen = rng(3)
    logits = torch.randn(6, 5000, generator=gen, device=DEV) * 3
    options = torch.tensor([0.7, 1.0, 0.0, 0.9, 1.3, 1.0], device=DEV), ints([0, 40, 5, 0, 600, 0]), torch.tensor([0.9, 0.8, 1.0, 1.0, 0.95, 0.5], device=DEV)
    probs, tokens, parents, q_start, u, draft = drafted_step(300, [6, 1, 30, 12], "tree", True, 4)
    u = torch.tensor(u, device=DEV)
    verified = ([ints(v) if isinstance(v, (list, tuple)) else v for v in (tokens, parents, q_start)])
    cache = torch.randn(2, 20, 2, 16, 24, generator=gen, device=DEV)
    nodes, table = ints([[0, 2, 5, 9], [0, 1, 4, -1]]), ints([list(range(10)), list(range(10, 20))])
    return logits, options, probs, verified, u, draft, cache, nodes, table


class Tail:
    def __init__(self, ops):
        self.ops = ops
        self.logits, self.options, self.probs, self.verified, self.u, self.draft, self.cache, self.nodes, self.table = last_steps()
        S = self.verified[2].numel() - 1
        self.layers = ops.CacheLayers([(self.cache[0], self.cache[1])])
        self.starts, self.accepted = ints([20, 33]), ints([3, 2])
        self.out = [torch.zeros_like(self.logits), ints([[0] * 8] * S), ints([0] * S), ints([0] * S)]
        self.before = self.cache.clone()

    def reset(self):
        for t in self.out:
            t.zero_()
        self.cache.copy_(self.before)

    def run(self):
        self.ops.sampling_probs(self.logits, self.out[0], *self.options)
        self.ops.verify_tree(self.probs, *self.verified, self.u, *self.out[1:], draft_probs=self.draft)
        self.ops.keep_tree_rows(self.layers, self.table, self.starts, self.nodes, self.accepted)

    def left(self):
        torch.cuda.synchronize()
        return [t.clone() for t in self.out] + [self.cache.clone()]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_bits_on_another_stream_and_recorded(ops):
    tail = Tail(ops)
    tail.run()
    want = tail.left()
    assert not torch.equal(want[-1], tail.before) and want[2].sum() > 0
    for _ in range(3):
        tail.reset()
        tail.run()
        assert same(tail.left(), want)
    tail.reset()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tail.run()
    assert same(tail.left(), want)
    tail.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tail.run()
    for _ in range(3):
        tail.reset()
        graph.replay()
        assert same(tail.left(), want)


def test_two_threads_at_once(ops):
    """Each with inputs, a workspace and a stream of its own."""
    from ferrisinfer_b200.engine.workspace import Workspace

    shapes = [([9] * 6, [700] * 6), ([40], [3000])]
    work = []
    for i, (nodes, starts) in enumerate(shapes):
        step, workspace, tail = Step(torch.bfloat16, 14, 2, 64, 16, nodes, starts, seed=3 + i), Workspace(DEV), Tail(ops)
        want = step.run(ops, workspace).clone()
        tail.run()
        work.append((step, workspace, tail, want, tail.left()))
    wrong = []

    def run(step, workspace, tail, want, left):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    tail.reset()
                    out = torch.zeros_like(want)
                    for _ in range(4):
                        ops.tree_attention(step.q, out, step.k, step.v, *step.device_tensors, *step.most, step.heads, step.D ** -0.5, workspace=workspace)
                    tail.run()
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(out, want) or not same([*tail.out, tail.cache], left):
                        wrong.append("values")
        except Exception as e:  # (said in the thread that waits)
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads, kv_heads, D, page_size", [(14, 2, 64, 16), (2, 1, 128, 16), (16, 1, 128, 32), (3, 1, 40, 7)])
@pytest.mark.parametrize("requests", [127, 128, 129, 333])
def test_attention_of_many_requests(ops, dtype, heads, kv_heads, D, page_size, requests):
    """Up to 128 requests are fetched once for a block's warps, more of them by every warp as it comes to them."""
    from ferrisinfer_b200.engine.workspace import Workspace

    draw = random.Random(requests)
    nodes = [draw.choice([0, 1, 2, 5, 17]) for _ in range(requests)]
    starts = [draw.choice([0, 1, 40, 129, 300]) for _ in range(requests)]
    starts[7], nodes[7] = 4000, 9
    step = Step(dtype, heads, kv_heads, D, page_size, nodes, starts, extra_columns=8)
    step.check(step.run(ops, Workspace(DEV)))
    step.check(step.run(ops, Workspace(DEV), window=33), window=33)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("window", [0, 100])
def test_rows_of_the_text_beyond_what_there_is(ops, dtype, window):
    """A request that says it has more rows than its table sees those that the table has, and behind a window none of them."""
    from ferrisinfer_b200.engine.workspace import Workspace

    step = Step(dtype, 12, 2, 64, 16, [5, 12], [60, 200])
    for start in (0x7fffffff, 1 << 30, 100000):
        step.starts[0] = start
        out = torch.full((17, 12 * 64), 7.0, dtype=dtype, device=DEV)
        ops.tree_attention(step.q, out, step.k, step.v, ints(step.tables), ints(step.q_start), ints(step.starts), ints(step.parents), 12, 212, 12, 0.125, window=window,
                           workspace=Workspace(DEV))
        if window:
            assert (out[:5] == 0).all()
        assert not (out[5:] == 7).any() and torch.isfinite(out[5:]).all()


def test_outputs_that_overlap_are_refused(ops):
    from ferrisinfer_b200.engine.workspace import Workspace
    from ferrisinfer_b200.errors import KernelError

    step = Step(torch.bfloat16, 4, 2, 64, 16, [3], [20])
    with pytest.raises(KernelError, match="overlap"):
        step.run(ops, Workspace(DEV), out=torch.zeros(1, 256, dtype=torch.bfloat16, device=DEV).expand(3, 256))
