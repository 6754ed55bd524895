"""Several conversations on one model over paged caches, with drafted tokens:
prompts in chunks beside single tokens, trees verified and their accepted rows
kept, every call as a program that serves them would make it. The tokens are the
oracle's greedy ones."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import ref
from titania_amd import QWEN3_TINY, TH_KV_BF16, TH_KV_F32, synth
from test_paged import rope_table

pytestmark = pytest.mark.gpu
CFG = QWEN3_TINY
PAGE, PAGES = 16, 24


class Serving:
    """The layers of CFG over paged caches, in the device's calls."""

    def __init__(self, hip, weights, kv):
        self.hip = hip
        w = {k: hip.upload(t) for k, t in weights.items()}
        self.layers = [[w[n] for n in synth.layer_names(i)] for i in range(CFG.num_hidden_layers)]
        self.table, self.norm = w["model.embed_tokens.weight"], w["model.norm.weight"]
        self.head = w.get("lm_head.weight", self.table)
        self.caches = [hip.alloc_paged(PAGES, PAGE, CFG.num_key_value_heads, CFG.head_dim(), kv) for _ in self.layers]
        self.batch = hip.alloc_batch(self.caches[0], CFG.num_attention_heads, 4, 128, PAGES)
        t = rope_table(PAGES * PAGE, CFG.head_dim(), CFG.rope_theta)
        self.rope = hip.alloc(t.size)
        hip.write(self.rope, t)

    def step(self, context, new, pages, tokens, parents=None):
        """The logits of a step's tokens."""
        hip, n, eps = self.hip, len(tokens), CFG.rms_norm_eps
        H, I, qd, kvd = CFG.hidden_size, CFG.intermediate_size, CFG.num_attention_heads * CFG.head_dim(), CFG.num_key_value_heads * CFG.head_dim()
        hip.set_batch(self.batch, context, new, [p for s in pages for p in s], parents)
        x, xb, y, q, k, v, gate, up = (hip.alloc(n * w) for w in (H, H, H, qd, kvd, kvd, I, I))
        out = hip.alloc(n * qd)
        hip.embed(x, self.table, tokens)
        add = None
        for (attn_norm, wq, wk, wv, wo, q_norm, k_norm, mlp_norm, wg, wu, wd), cache in zip(self.layers, self.caches):
            hip.add_rmsnorm(x, add, xb, attn_norm, eps)
            hip.matmul(q, wq, xb)
            hip.matmul(k, wk, xb)
            hip.matmul(v, wv, xb)
            hip.paged_append(q, q, k, v, q_norm, k_norm, self.rope, cache, self.batch, eps)
            hip.paged_attention(out, q, cache, self.batch)
            hip.matmul(y, wo, out)
            hip.add_rmsnorm(x, y, xb, mlp_norm, eps)
            hip.gate_up_silu(gate, up, wg, wu, xb)
            hip.matmul(y, wd, gate)
            add = y
        hip.add_rmsnorm(x, add, xb, self.norm, eps)
        logits = hip.alloc(n * CFG.vocab_size)
        hip.matmul(logits, self.head, xb)
        return logits


def draft(r, truth, at, n):
    """A tree after the token truth[at]: a branch of what comes next, cut at a
    wrong token, and others in between. Returns tokens and parents, the first
    of them truth[at]."""
    tokens, parents, on = [truth[at]], [-1], 0
    for i in range(1, n):
        if r.random() < 0.6 and on >= 0 and at + depth(parents, on) + 1 < len(truth):
            parents.append(on)
            tokens.append(truth[at + depth(parents, on) + 1])
            on = i if r.random() < 0.9 else -1
        else:
            parents.append(int(r.integers(0, i)))
            tokens.append(int(r.integers(0, CFG.vocab_size)))
    return tokens, parents


def depth(parents, i):
    d = 0
    while parents[i] >= 0:
        i, d = parents[i], d + 1
    return d


@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
def test_drafted_tokens_of_three_conversations(hip, kv):
    weights = synth.weights(CFG, seed=5, random_gains=True)
    oracle, r = ref.RefModel(CFG, weights), np.random.default_rng(4)
    steps = 24
    prompts = [synth.prompt(n, CFG.vocab_size, seed=n) for n in (37, 5, 70)]
    # Picks that the two largest logits decide: these are off by 1e-4 at most,
    # over bf16 caches by 2e-2.
    truths, decided = [], []
    for p in prompts:
        toks, gaps, _ = oracle.generate(oracle.state(len(p) + steps), p, steps)
        truths.append([int(t) for t in toks])
        decided.append(gaps > (2e-4 if kv == TH_KV_F32 else 4e-2))
    assert np.mean(decided) > 0.8
    m = Serving(hip, weights, kv)
    free = list(r.permutation(PAGES))
    pages, context = [[], [], []], [0, 0, 0]

    def grow(s, n):
        while len(pages[s]) * PAGE < context[s] + n:
            pages[s].append(free.pop())
        return pages[s][:-(-(context[s] + n) // PAGE)]

    # The prompts: the first and the last in chunks, beside the second's.
    fed = [0, 0, 0]
    while any(f < len(p) for f, p in zip(fed, prompts)):
        new = [min(n, len(p) - f) for n, f, p in zip((20, 5, 41), fed, prompts)]
        tokens = np.concatenate([p[f:f + n] for p, f, n in zip(prompts, fed, new)])
        logits = m.step(context, new, [grow(s, n) for s, n in enumerate(new)], tokens)
        picks, _, _ = hip.accept(m.batch, logits, tokens)
        for s, n in enumerate(new):
            if n:
                last = int(picks[sum(new[:s + 1]) - 1])
                context[s] += n
                fed[s] += n
                if fed[s] == len(prompts[s]):
                    assert last == truths[s][0] or not decided[s][0]
    # Drafts of the three at once, of the first two alone, ...
    said = [0, 0, 0]  # of each the place of its next token
    taken = 0
    for turn in range(200):
        if min(said) >= steps - 1:
            break
        who = [s for s in range(3) if said[s] < steps - 1 and (turn % 3 or s != 2)]
        if not who:
            continue
        trees = {s: draft(r, truths[s], said[s], int(r.integers(1, 14))) for s in who}
        new = [len(trees[s][0]) if s in trees else 0 for s in range(3)]
        tokens = [t for s in who for t in trees[s][0]]
        logits = m.step(context, new, [grow(s, n) for s, n in enumerate(new)], tokens, [p for s in who for p in trees[s][1]])
        picks, n_kept, kept = hip.accept(m.batch, logits, tokens)
        hip.paged_keep(m.caches, m.batch, n_kept, kept)
        for s in who:
            first, path = sum(new[:s]), kept[sum(new[:s]):][:n_kept[s]]
            assert [tokens[first + i] for i in path] == truths[s][said[s]:said[s] + len(path)]
            after = said[s] + len(path)
            if after < steps and decided[s][after]:
                assert int(picks[first + path[-1]]) == truths[s][after]
            taken += len(path) - 1
            context[s] += len(path)
            said[s] = after
    assert min(said) >= steps - 1 and taken > 10
