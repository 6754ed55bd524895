"""Work of a program that serves several conversations at once, and drafts
tokens ahead of the model, as cases to be timed and compared: keys and values
in a paged cache, written and read for a batch of sequences.

A sequence s has context[s] positions in the cache and new[s] tokens of this
step, at the positions behind them, in pages[s]: position p lies in row
p % page of its page p // page. The new tokens are a chain, or a tree: token i
then follows token parent[i] < i (or the context, -1), has its depth's
rotation and sees the context, its ancestors and itself. Four operators:

- "append": queries and keys normalised for each head and rotated, keys and
  values written to their rows of the cache;
- "attention": of the new tokens over the cache, causal, or along the tree;
- "accept": the greedy verification of drafted tokens: each token's largest
  logit, and the path from token 0 on, to the first child whose token that is;
- "keep": the rows of the tokens that were accepted, moved up behind the
  context, in every layer's cache.

Heads are those of the Qwen3-0.6B (16 and 8 of 128) and Qwen3-4B (32 and 8)
layers, activations f32, caches f32 or bf16.

The framework's calls go to its device's own stream, which neither waits for
torch's streams nor is waited for by them. What `prepare` writes with torch is
there when it returns; a pass of the framework's calls is over, and its outputs
may be read, once the whole device has been waited for
(`torch.cuda.synchronize()`): an event on a torch stream does not see it.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # Decode: a conversation's first tokens, where only latency counts, and
        # one token after a long document.
        {"name": "token", "kind": "attention", "kv": "f32", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16,
         "seqs": 1, "least": 40, "most": 40, "new": 1, "tree": False},
        {"name": "long token", "kind": "attention", "kv": "f32", "heads": 16, "kv_heads": 8, "dim": 128, "page": 64,
         "seqs": 1, "least": 32767, "most": 32767, "new": 1, "tree": False},
        # Decode of many conversations of all lengths in one step.
        {"name": "batch", "kind": "attention", "kv": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "seqs": 64, "least": 120, "most": 8000, "new": 1, "tree": False},
        # Chunks of three prompts, one of them from its start.
        {"name": "chunks", "kind": "attention", "kv": "f32", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "seqs": 3, "least": 0, "most": 5000, "new": 2048, "tree": False},
        # A tree of 60 drafted tokens after a long document.
        {"name": "tree", "kind": "attention", "kv": "f32", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "seqs": 1, "least": 12001, "most": 12001, "new": 60, "tree": True},
        # Trees of up to 25 tokens of a dozen conversations.
        {"name": "trees", "kind": "attention", "kv": "bf16", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16,
         "seqs": 12, "least": 300, "most": 4000, "new": 25, "tree": True},
        # A layer's append, decoding and over the chunks of long prompts.
        {"name": "append token", "kind": "append", "kv": "f32", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16,
         "seqs": 1, "least": 40, "most": 40, "new": 1, "tree": False},
        {"name": "append prompt", "kind": "append", "kv": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "seqs": 5, "least": 0, "most": 2000, "new": 2048, "tree": False},
        # Verification over the vocabulary: one tree, and a batch of them.
        {"name": "accept", "kind": "accept", "seqs": 1, "new": 24, "vocab": 151936},
        {"name": "accept batch", "kind": "accept", "seqs": 16, "new": 40, "vocab": 151936},
        # The accepted rows in the caches of all layers.
        {"name": "keep", "kind": "keep", "kv": "f32", "kv_heads": 8, "dim": 128, "page": 16, "seqs": 1, "least": 40,
         "most": 40, "new": 24, "layers": 28},
        {"name": "keep batch", "kind": "keep", "kv": "bf16", "kv_heads": 8, "dim": 128, "page": 32, "seqs": 24,
         "least": 20, "most": 90, "new": 30, "layers": 36},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


# The listed attentions' most pairs of tokens, and positions of a batch.
MOST_PAIRS, MOST_POSITIONS = 18_000_000, 250_000


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "append", "accept", "keep"])
    if kind == "accept":
        seqs = _log_int(rng, 1, 16)
        return {"kind": kind, "seqs": seqs, "new": _log_int(rng, 1, 40), "vocab": rng.choice([151936, _log_int(rng, 100, 151936)])}
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (4, 2), (8, 8), (8, 1)])
    case = {"kind": kind, "kv": rng.choice(["f32", "bf16"]), "heads": heads, "kv_heads": kv_heads, "dim": 128,
            "page": rng.choice([16, 32, 64, 128])}
    if kind == "keep":
        del case["heads"]
        most = _log_int(rng, 1, 90)
        return case | {"seqs": _log_int(rng, 1, 24), "least": rng.randint(0, most), "most": most, "new": _log_int(rng, 1, 40),
                       "layers": rng.randint(1, 36)}
    tree = rng.random() < 0.4
    seqs = _log_int(rng, 1, 64)
    new = rng.choice([1, _log_int(rng, 1, 64)]) if tree or rng.random() < 0.6 else _log_int(rng, 1, 2048)
    new = min(new, max(1, 6000 // seqs)) if kind == "append" else new
    most = _log_int(rng, 1, 32767)
    if kind == "attention":
        most = max(1, min(most, MOST_POSITIONS // seqs, MOST_PAIRS // (seqs * new)))
        while seqs * new * (most + new) > MOST_PAIRS and new > 1:
            new = max(1, new // 2)
    else:
        most = min(most, 4000)
    return case | {"seqs": seqs, "least": rng.randint(0, most), "most": most, "new": new, "tree": tree}


# ---- a step's batch: the same for every seed, but for the pages' order ----

class Step:
    """The sequences of a case: contexts, new tokens, trees, positions and rows."""

    def __init__(self, case):
        rng = random.Random(case["seqs"] * 1009 + case["new"])
        seqs, least, most = case["seqs"], case.get("least", 0), case.get("most", 0)
        self.context = [least + (most - least) * i // max(1, seqs - 1) for i in range(seqs)]
        rng.shuffle(self.context)
        # The first has the most new tokens, the others from half as many on.
        self.new = [case["new"] if i == 0 else rng.randint((case["new"] + 1) // 2, case["new"]) for i in range(seqs)]
        self.first = [sum(self.new[:i]) for i in range(seqs)]
        self.tokens = sum(self.new)
        self.tree = case.get("tree", True)
        self.parents, self.depth = [], []
        for n in self.new:
            parent = [i - 1 if not self.tree or i == 0 else rng.randint(max(0, i - 6), i - 1) for i in range(n)]
            depth = []
            for p in parent:
                depth.append(depth[p] + 1 if p >= 0 else 0)
            self.parents += parent
            self.depth += depth
        page = case.get("page", 16)
        self.n_pages = [-(-(c + n) // page) for c, n in zip(self.context, self.new)]

    def seen(self):
        """(query token, key) pairs of the step."""
        return sum(c * n + (sum(self.depth[f:f + n]) + n) for c, n, f in zip(self.context, self.new, self.first))

    def plan(self, case, seed):
        """What a program keeps of a step on the GPU, as index tensors."""
        page, most_new = case.get("page", 16), max(self.new)
        total = sum(self.n_pages)
        order = np.random.RandomState(seed % (1 << 31)).permutation(total)
        table, at, pages = np.zeros((len(self.new), max(self.n_pages)), np.int64), 0, []
        for s, n in enumerate(self.n_pages):
            table[s, :n] = order[at:at + n]
            pages += list(order[at:at + n])
            at += n
        seq = np.repeat(np.arange(len(self.new)), self.new)
        index = np.arange(self.tokens) - np.repeat(self.first, self.new)
        slot = np.repeat(self.context, self.new) + index
        parents = np.array(self.parents, np.int64)
        ancestors = np.zeros((len(self.new), most_new, most_new), bool)
        for s, (f, n) in enumerate(zip(self.first, self.new)):
            if not self.tree:
                ancestors[s, :n, :n] = np.tri(n, dtype=bool)
                continue
            for i in range(n):
                if parents[f + i] >= 0:
                    ancestors[s, i] = ancestors[s, parents[f + i]]
                ancestors[s, i, i] = True
        d = {"table": table, "seq": seq, "index": index, "parents": parents, "ancestors": ancestors,
             "position": np.repeat(self.context, self.new) + np.array(self.depth), "context": np.array(self.context),
             "page": table[seq, slot // page], "row": slot % page}
        return {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in d.items()}, np.array(pages, np.uint32)


# ---- what a program has in hand ----

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(g, case, pages):
    """A cache's pages: [page][keys, values][head][row][dim]."""
    p = torch.randn((pages, 2, case["kv_heads"], case["page"], case["dim"]), generator=g, device="cuda")
    return p.to(torch.bfloat16) if case["kv"] == "bf16" else p


def _inputs(case, seed):
    """The case's tensors, of either side."""
    g, step = _generator(seed), Step(case)
    if case["kind"] == "accept":
        logits = 4 * torch.randn((step.tokens, case["vocab"]), generator=g, device="cuda")
        # Two drafted tokens of three are the model's own choice after their parent.
        first = torch.tensor(np.repeat(step.first, step.new), device="cuda")
        parents = torch.tensor(step.parents, device="cuda")
        choice = logits.argmax(1)[first + parents.clamp_min(0)]
        other = torch.randint(0, case["vocab"], (step.tokens,), generator=g, device="cuda")
        right = torch.rand(step.tokens, generator=g, device="cuda") < 0.67
        return {"logits": logits, "tokens": torch.where(right, choice, other)}
    pages = sum(step.n_pages)
    if case["kind"] == "keep":
        pools = [_pool(g, case, pages) for _ in range(case["layers"])]
        # Paths down the trees: of each, one to all of a random token's ancestors.
        r, kept = random.Random(seed), []
        for f, n in zip(step.first, step.new):
            at, path = r.randrange(n), []
            while at >= 0:
                path.append(at)
                at = step.parents[f + at]
            kept.append(path[::-1])
        return {"pools": pools, "kept": kept}
    pool, dim = _pool(g, case, pages), case["dim"]
    if case["kind"] == "attention":
        # Queries and keys as the head norms leave them: about sqrt(dim) long.
        return {"pool": pool, "q": torch.randn((step.tokens, case["heads"], dim), generator=g, device="cuda")}
    shape = lambda heads: (step.tokens, heads, dim)  # noqa: E731
    q, k, v = (torch.randn(shape(h), generator=g, device="cuda") * s for h, s in ((case["heads"], 2.0), (case["kv_heads"], 3.0), (case["kv_heads"], 0.5)))
    gains = [(1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(torch.bfloat16) for _ in range(2)]
    most = max(c + n for c, n in zip(step.context, step.new))
    freq = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * freq
    rope = torch.stack([angle.cos(), angle.sin()], -1).float()
    return {"pool": pool, "q": q, "k": k, "v": v, "q_gain": gains[0], "k_gain": gains[1], "rope": rope}


_device = None


def _hip():
    global _device
    if _device is None:
        from titania_amd.device import Hip

        _device = Hip(0)
    return _device


class _InPlace:
    """A handle's memory, for torch to look at in place (which keeps the
    handle): a handle points at the device address first."""

    def __init__(self, held, shape: tuple, typestr: str):
        self.held = held
        address = ctypes.c_void_p.from_address(held.handle).value
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (address, False), "version": 2}


def _view(buf, *shape) -> torch.Tensor:
    """A buffer's values where they are: a program that chains operations
    reads none of them back."""
    return torch.as_tensor(_InPlace(buf, shape, "<f4"), device="cuda")


def _buffer(values: torch.Tensor):
    b = _hip().alloc(values.numel())
    _view(b, values.numel()).copy_(values.reshape(-1))
    return b


def _gains(values: torch.Tensor):
    from titania_amd.device import Tensor

    return _hip().upload(Tensor(tuple(values.shape), values.view(torch.int16).cpu().numpy().view("uint16")))


def _cache(case, pool: torch.Tensor):
    """A paged cache that holds `pool`, and its memory as a tensor."""
    from titania_amd import TH_KV_BF16, TH_KV_F32

    bf16 = case["kv"] == "bf16"
    c = _hip().alloc_paged(pool.shape[0], case["page"], case["kv_heads"], case["dim"], TH_KV_BF16 if bf16 else TH_KV_F32)
    seen = torch.as_tensor(_InPlace(c, tuple(pool.shape), "<i2" if bf16 else "<f4"), device="cuda")
    seen = seen.view(torch.bfloat16) if bf16 else seen
    seen.copy_(pool)
    return c, seen


def prepare(case, seed):
    step, x = Step(case), _inputs(case, seed)
    plan, pages = step.plan(case, seed)
    state = {"case": case, "plan": plan, "step": step}
    if not own:
        if case["kind"] == "keep":
            flat = [(s, j, i) for s, path in enumerate(x["kept"]) for j, i in enumerate(path)]
            state["moves"] = torch.tensor(flat, device="cuda").T
        torch.cuda.synchronize()
        return state | x
    hip = _hip()
    kv = case if "kv" in case else {"kv": "f32", "kv_heads": 1, "dim": 64, "page": 16}
    caches = [_cache(kv, p) for p in (x["pools"] if "pools" in x else [x["pool"]] if "pool" in x
                                      else [torch.zeros((sum(step.n_pages), 2, 1, 16, 64), device="cuda")])]
    state["caches"], state["seen"] = [c for c, _ in caches], [t for _, t in caches]
    batch = hip.alloc_batch(state["caches"][0], case.get("heads", kv["kv_heads"]), len(step.new), step.tokens, len(pages))
    hip.set_batch(batch, step.context, step.new, pages, step.parents if step.tree else None)
    state["batch"] = batch
    if case["kind"] == "accept":
        state["logits"], state["tokens"] = _buffer(x["logits"]), x["tokens"].cpu().numpy().astype(np.uint32)
    elif case["kind"] == "keep":
        kept = np.full(step.tokens, -1, np.int32)
        for f, path in zip(step.first, x["kept"]):
            kept[f:f + len(path)] = path
        state["n_kept"], state["kept"] = np.array([len(p) for p in x["kept"]], np.uint32), kept
    else:
        state["q"], state["out"] = _buffer(x["q"]), hip.alloc(x["q"].numel())
        state["seen_out"] = _view(state["out"], *x["q"].shape)
        if case["kind"] == "append":
            state |= {n: _buffer(x[n]) for n in ("k", "v", "rope")} | {n: _gains(x[n]) for n in ("q_gain", "k_gain")}
    torch.cuda.synchronize()  # the device's own stream does not wait for torch's
    return state


# ---- a pass ----

def _attention(state):
    case, plan, q, pool = state["case"], state["plan"], state["q"], state["pool"]
    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    group = heads // kv_heads
    seqs, most_new = plan["ancestors"].shape[:2]
    length = plan["table"].shape[1] * page
    kv = pool[plan["table"]].float()  # [seq][page][2][head][row][dim]
    keys, values = (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, length, dim) for i in (0, 1))
    rows = torch.zeros((seqs, most_new, heads, dim), device="cuda")
    rows[plan["seq"], plan["index"]] = q
    rows = rows.view(seqs, most_new, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    scores = torch.matmul(rows, keys.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(dim))
    # A key is seen from the context, or as an ancestor.
    at = torch.arange(length, device="cuda")[None] - plan["context"][:, None]
    drafted = plan["ancestors"].gather(2, at.clamp(0, most_new - 1)[:, None].expand(seqs, most_new, length))
    hidden = ~((at < 0)[:, None] | (drafted & (at < most_new)[:, None]))
    scores.view(seqs, kv_heads, group, most_new, length).masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(scores, values) / scores.sum(-1, keepdim=True)
    out = out.view(seqs, kv_heads, group, most_new, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most_new, heads, dim)
    return out[plan["seq"], plan["index"]]


def _normed_and_rotated(x, gain, rope):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()
    a, b = x.chunk(2, -1)
    cos, sin = rope[:, None, :, 0], rope[:, None, :, 1]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(state):
    plan, pool = state["plan"], state["pool"]
    rope = state["rope"][plan["position"]]
    pool[plan["page"], 0, :, plan["row"]] = _normed_and_rotated(state["k"], state["k_gain"], rope).to(pool.dtype)
    pool[plan["page"], 1, :, plan["row"]] = state["v"].to(pool.dtype)
    return {"q": _normed_and_rotated(state["q"], state["q_gain"], rope), "cache": pool}


def _accept(state):
    plan, tokens = state["plan"], state["tokens"]
    seq, index, parents = plan["seq"], plan["index"], plan["parents"]
    pick = state["logits"].argmax(1)
    first = torch.arange(len(seq), device="cuda") - index
    # A child of its parent's choice that has no lower such brother.
    fits = (parents >= 0) & (tokens == pick[first + parents.clamp_min(0)])
    seqs, most = plan["ancestors"].shape[:2]
    brothers = torch.full((seqs, most), most, device="cuda")
    brothers.view(-1).scatter_reduce_(0, seq * most + parents.clamp_min(0), torch.where(fits, index, most), "amin")
    fits = (fits & (brothers[seq, parents.clamp_min(0)] == index)) | (index == 0)
    miss = torch.zeros((seqs, most), device="cuda")
    miss[seq, index] = (~fits).float()
    kept = (torch.matmul(plan["ancestors"].float(), miss[:, :, None])[:, :, 0] == 0)[seq, index]
    n_kept = torch.zeros(seqs, dtype=torch.int64, device="cuda").scatter_add_(0, seq, kept.long())
    place = kept.long().cumsum(0) - 1
    before = n_kept.cumsum(0) - n_kept
    path = torch.full_like(index, -1)
    at = torch.where(kept, first + place - before[seq], len(seq))
    path = torch.cat([path, path[:1]]).scatter_(0, at, torch.where(kept, index, -1))[:-1]
    return {"picks": pick, "n_kept": n_kept, "kept": path}


def _keep(state):
    (seq, to, at), plan, page = state["moves"], state["plan"], state["case"]["page"]
    source, target = plan["context"][seq] + at, plan["context"][seq] + to
    source, target = ((plan["table"][seq, p // page], p % page) for p in (source, target))
    for pool in state["pools"]:
        rows = pool.transpose(2, 3)  # [page][2][row][head][dim]
        rows[target[0], :, target[1]] = rows[source[0], :, source[1]]
    return state["pools"]


def _own(state):
    case, hip, batch = state["case"], _hip(), state["batch"]
    if case["kind"] == "attention":
        hip.paged_attention(state["out"], state["q"], state["caches"][0], batch)
        return state["seen_out"]
    if case["kind"] == "append":
        hip.paged_append(state["out"], state["q"], state["k"], state["v"], state["q_gain"], state["k_gain"], state["rope"],
                         state["caches"][0], batch, EPS)
        return {"q": state["seen_out"], "cache": state["seen"][0]}
    if case["kind"] == "accept":
        picks, n_kept, kept = hip.accept(batch, state["logits"], state["tokens"])
        return {"picks": picks.astype(np.int64), "n_kept": n_kept.astype(np.int64), "kept": kept.astype(np.int64)}
    hip.paged_keep(state["caches"], batch, state["n_kept"], state["kept"])
    return state["seen"]


def run(state):
    if own:
        return _own(state)
    return {"attention": _attention, "append": _append, "accept": _accept, "keep": _keep}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----

def work(case):
    step = Step(case)
    if case["kind"] == "accept":
        return {"bytes": 4 * step.tokens * case["vocab"], "flops": step.tokens * case["vocab"]}
    size = 4 if case["kv"] == "f32" else 2
    row = 2 * case["kv_heads"] * case["dim"] * size  # a position's keys and values
    if case["kind"] == "keep":  # a path is about as long as the trees are deep
        return {"bytes": 2 * case["layers"] * row * sum(max(step.depth[f:f + n]) + 1 for f, n in zip(step.first, step.new)), "flops": 0}
    values = step.tokens * case["heads"] * case["dim"]
    if case["kind"] == "append":
        new = step.tokens * case["kv_heads"] * case["dim"]
        return {"bytes": 8 * values + 8 * new + step.tokens * (row + 4 * case["dim"]), "flops": 8 * (values + new)}
    positions = sum(c + n for c, n in zip(step.context, step.new))
    return {"bytes": 8 * values + row * positions, "flops": 4 * case["heads"] * case["dim"] * step.seen()}


# ---- the same in 64 bits ----

def exact(case, seed):
    step, x = Step(case), _inputs(case, seed)
    plan, _ = step.plan(case, seed)
    if case["kind"] == "accept":
        return None  # whole numbers
    if case["kind"] == "keep":
        pools = [p.double() for p in x["pools"]]
        for s, (c, path) in enumerate(zip(step.context, x["kept"])):
            places = [(int(plan["table"][s, p // case["page"]]), p % case["page"]) for p in range(c, c + step.new[s])]
            for pool in pools:
                moved = [pool[places[i][0], :, :, places[i][1]].clone() for i in path]
                for (page, row), values in zip(places, moved):
                    pool[page, :, :, row] = values
        return pools
    dim = case["dim"]
    if case["kind"] == "append":
        table, where = x["rope"].double()[plan["position"]], (plan["page"], plan["row"])
        turn = torch.complex(table[..., 0], table[..., 1])[:, None]

        def rotated(v, gain):
            v = v.double()
            v = v * gain.double() / torch.sqrt((v * v).sum(-1, keepdim=True) / dim + EPS)
            z = torch.complex(v[..., :dim // 2], v[..., dim // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        cache = x["pool"].double().permute(0, 3, 1, 2, 4).contiguous()  # [page][row][2][head][dim]
        cache[where] = torch.stack([rotated(x["k"], x["k_gain"]), x["v"].double()], 1)
        return {"q": rotated(x["q"], x["q_gain"]), "cache": cache.permute(0, 2, 3, 1, 4).contiguous()}
    out = torch.empty((step.tokens, case["heads"], dim), dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for s, (c, n, f, pages) in enumerate(zip(step.context, step.new, step.first, step.n_pages)):
        held = x["pool"][plan["table"][s, :pages]].double().permute(1, 2, 0, 3, 4).reshape(2, case["kv_heads"], -1, dim)[:, :, :c + n]
        sees = torch.cat([torch.ones((n, c), dtype=torch.bool, device="cuda"), plan["ancestors"][s, :n, :n]], 1)
        for h in range(case["heads"]):
            k, v = held[0, h // group], held[1, h // group]
            score = torch.mm(x["q"][f:f + n, h].double(), k.t()) / math.sqrt(dim)
            out[f:f + n, h] = torch.mm(torch.softmax(score.masked_fill(~sees, -math.inf), 1), v)
    return out
