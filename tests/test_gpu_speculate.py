"""Speculative steps of the engine (sdy_engine_speculate): drafted trees evaluated in one pass give the tokens, the cache and
the logits that one token at a time gives, whatever is drafted."""
import numpy as np
import pytest

from conftest import engine_env
from sardyne_amd.engine import LoadedModel, greedy
from sardyne_amd.gguf_synth import write_model
from test_gpu_engine import SPECS

pytestmark = pytest.mark.gpu

PROMPT = [3, 14, 15, 9, 26, 5, 35]
USED = ["qwen2-kquant", "qwen2-q0", "llama-kquant", "moe-kquant", "qwen2-gqa8-hd128", "moe-16x4-ffn768", "qwen2-kquant-v4k"]


@pytest.fixture(scope="module", params=USED)
def model(request, tmp_path_factory):
    p = tmp_path_factory.mktemp("spec") / "m.gguf"
    write_model(p, SPECS[request.param], seed=11)
    with LoadedModel(p) as m:
        yield m


def draft(right, vocab, rng, n):
    """A tree under the context's next token with the right continuation among wrong ones: tokens and parents."""
    tokens, parents, last = [], [], -1
    for tok in right:
        for _ in range(int(rng.integers(0, 3))):
            if last >= 0:  # a wrong sibling, sometimes with a child
                tokens.append(int((tok + 1 + rng.integers(0, vocab - 1)) % vocab))
                parents.append(last)
                if rng.random() < 0.5:
                    tokens.append(int(rng.integers(0, vocab)))
                    parents.append(len(tokens) - 2)
        tokens.append(int(tok))
        parents.append(last)
        last = len(tokens) - 1
    return tokens[:n], parents[:n]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("right", [0, 2, 6])
def test_greedy_speculation_gives_the_greedy_tokens(model, kv, right):
    rng = np.random.default_rng(right)
    with engine_env(SARDYNE_KV=kv):
        plain, spec = model.session(max_seq=48, n_batch=16), model.session(max_seq=48, n_batch=16)
    want = greedy(plain, PROMPT, 24)
    logits = plain.step(want[-1])  # position 31: after 24 tokens
    nxt = int(np.argmax(spec.feed(PROMPT)))
    got, steps = [], 0
    while len(got) < 24:
        assert nxt == want[len(got)]
        ahead = want[len(got):len(got) + 1 + right]
        tokens, parents = draft(ahead, model.n_vocab, rng, 16)
        before = spec.position
        path, nxt = spec.speculate(tokens, parents)
        assert path[0] == 0 and spec.position == before + len(path)
        got += [tokens[i] for i in path]
        steps += 1
    assert got[:24] == want
    assert steps <= 24 // (1 + min(right, 3)) + 2
    # the cache that the trees left: the next plain step's logits
    spec.rewind(len(PROMPT) + 23)
    again = spec.step(want[-1])
    assert np.abs(again - logits).max() <= 2e-4 * max(1.0, np.abs(logits).max()) * (1 if kv == "f32" else 8)


@pytest.mark.parametrize("how", [dict(temp=0.8), dict(temp=1.2, top_k=20, top_p=0.9), dict(temp=1.0, min_p=0.05)])
def test_sampled_speculation_gives_the_tokens_of_one_at_a_time(model, how):
    """One uniform number per position, the same for every node there."""
    rng = np.random.default_rng(5)
    u = rng.random(64).astype(np.float32)
    one, tree = model.session(max_seq=48, n_batch=16), model.session(max_seq=48, n_batch=16)
    first = int(np.argmax(one.feed(PROMPT)))
    want, nxt = [], first
    while len(want) < 20:
        want.append(nxt)
        path, nxt = one.speculate([nxt], [-1], u[one.position:one.position + 1], **how)
        assert path == [0]
    tree.feed(PROMPT)
    got, nxt = [], first
    while len(got) < 20:
        tokens, parents = draft(want[len(got):len(got) + 5], model.n_vocab, rng, 16)
        depth = []
        for p in parents:
            depth.append(depth[p] + 1 if p >= 0 else 0)
        path, nxt = tree.speculate(tokens, parents, u[tree.position + np.array(depth)], **how)
        got += [tokens[i] for i in path]
    assert got[:20] == want


def test_a_full_context_ends_the_path(model):
    s = model.session(max_seq=10, n_batch=16)
    nxt = int(np.argmax(s.feed(PROMPT)))
    want = greedy(model.session(max_seq=48), PROMPT, 8)
    path, after = s.speculate(want[:8], list(range(-1, 7)))
    assert nxt == want[0] and path == [0, 1, 2] and s.position == 10 and after == want[3]
    with pytest.raises(ValueError, match="contesto pieno"):
        s.speculate([1], [-1])
    s.clear()
    assert int(np.argmax(s.feed(PROMPT))) == nxt
    assert s.speculate([nxt], [-1])[1] == want[1]


@pytest.mark.parametrize("tokens,parents,match", [
    ([], [], "nessun token"), ([5], [0], "parents"), ([5, 6], [-1, -1], "parents"), ([5, 6], [-1, 1], "parents"),
    ([5, 6, 7], [-1, 0, -2], "parents"), ([300], [-1], "vocabolario"), ([5, -1], [-1, 0], "vocabolario"),
    ([5] * 9, [-1] + [0] * 8, "n=9"), ([5, 6], [-1], "parents")])
def test_refusals_leave_the_context(model, tokens, parents, match):
    s = model.session(max_seq=32, n_batch=8)
    s.feed(PROMPT)
    with pytest.raises(ValueError, match=match):
        s.speculate(tokens, parents)
    assert s.position == len(PROMPT)


def test_head_dim_32_is_refused(tmp_path):
    write_model(tmp_path / "m.gguf", SPECS["qwen3-q8"], seed=1)
    with LoadedModel(tmp_path / "m.gguf") as m:
        s = m.session(max_seq=32)
        s.feed(PROMPT)
        with pytest.raises(ValueError, match="head_dim"):
            s.speculate([1], [-1])


def test_between_plain_steps_and_prompts(model):
    """Speculative steps, recorded one-token steps and prompts in turn on one context."""
    want = greedy(model.session(max_seq=48), PROMPT, 16)
    s = model.session(max_seq=48, n_batch=16)
    assert int(np.argmax(s.feed(PROMPT))) == want[0]
    path, nxt = s.speculate(want[:4], [-1, 0, 1, 2])
    assert path == [0, 1, 2, 3] and nxt == want[4]
    for k in range(4, 8):
        nxt = int(np.argmax(s.step(nxt)))
        assert nxt == want[k + 1]
    path, nxt = s.speculate([want[8], want[9], 0], [-1, 0, 0])
    assert [want[8:10][i] for i in path] == want[8:10] and nxt == want[10]
    assert int(np.argmax(s.feed(want[10:13]))) == want[13]
    path, nxt = s.speculate([want[13]], [-1])
    assert nxt == want[14]
