"""The operators for sequences that share their beginnings, as cases that a program times.

Two kinds of work. Attention over the paged cache for a batch whose sequences hold the same pages at their front: several
continuations of one prompt, many questions behind one system prompt, or both, nested; one token each or runs of tokens. And
the copies that such sharing needs: the partly filled last page of a sequence that is forked, the fixed-size states of its
slot, and the pages that move when a cache is compacted into a new storage.

Attention of row t (sequence b, position p) and query head h, whose key/value head is g = h // (H / G), over keys j <= p that
lie in page table[b, j // 64]: s_j = scale * (q . k_j), with a cap c * tanh(s_j / c); softmax over j, with a sink's exp(sink[h])
in the denominator; sum of p_j v_j. A copy of pages: dst[unit, d, head, i] = src[unit, s, head, i] for i < rows and every pair
of page ids (s, d). A copy of slots: dst[d] = src[s] of every tensor.

Sizes are those of the repository's benchmark models (widths of heads, heads, key/value heads, layers) or lie around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _attn(seqs, prefix, private, tokens=1, groups=0, group_prefix=0, heads=32, kv=8, dim=64, vdim=None, cap=0.0, sink=False,
          dtype="bfloat16", name=None):
    """`seqs` sequences whose first `prefix` positions are the same; with `groups`, sequences i, i + groups, ... share another
    `group_prefix` behind them. Each holds up to `private` positions of its own, and brings up to `tokens` new ones."""
    c = {"op": "attention", "seqs": seqs, "prefix": prefix, "private": private, "tokens": tokens, "groups": groups,
         "group_prefix": group_prefix, "heads": heads, "kv": kv, "dim": dim, "vdim": vdim or dim, "cap": cap, "sink": sink, "dtype": dtype}
    return {"name": name, **c} if name else c


def _pages(pairs, rows, units, heads, dim, vdim=None, fork=False, dtype="bfloat16", name=None):
    """`pairs` copied pages of `units` cache units; `fork`: all from one page, into the same storage; else each from another, into
    another storage. `rows`: positions of a page that are copied (0: a different number for every pair)."""
    c = {"op": "pages", "pairs": pairs, "rows": rows, "units": units, "heads": heads, "dim": dim, "vdim": vdim or dim, "fork": fork,
         "dtype": dtype}
    return {"name": name, **c} if name else c


def _slots(pairs, units, state, conv, name=None):
    """`pairs` slots copied from one: in every unit a float32 state of `state` elements and bfloat16 rows of `conv` elements."""
    c = {"op": "slots", "pairs": pairs, "units": units, "state": state, "conv": conv}
    return {"name": name, **c} if name else c


def listed():
    return [
        # two continuations of a short prompt, a small model: latency is all
        _attn(2, 200, 5, heads=16, kv=4, dim=64, name="decode-b2-short"),
        # eight continuations of the headline's context, its head layout (every head has keys of its own)
        _attn(8, 4096, 150, heads=32, kv=32, dim=64, name="decode-b8-4k"),
        # a full batch behind one long system prompt, grouped heads of 128, answers of unequal lengths
        _attn(64, 8192, 300, heads=32, kv=8, dim=128, name="decode-b64-8k-h128"),
        # six prompts behind a common one, eight samples of each; capped scores and sinks
        _attn(48, 1500, 400, groups=6, group_prefix=700, heads=16, kv=4, dim=64, vdim=128, cap=30.0, sink=True, name="decode-groups-cap-sink"),
        # the 32-bit engine: a small batch behind a prompt
        _attn(12, 1000, 70, heads=32, kv=8, dim=64, dtype="float32", name="decode-b12-f32"),
        # questions of a few to ninety tokens behind a system prompt, all in one prompt step
        _attn(16, 4001, 30, tokens=90, heads=32, kv=8, dim=64, name="prompt-b16-4k"),
        # many short questions behind a very long document
        _attn(64, 16384, 0, tokens=40, heads=32, kv=8, dim=128, name="prompt-b64-16k-h128"),
        # the same in 32-bit, small
        _attn(5, 600, 10, tokens=33, heads=16, kv=4, dim=64, dtype="float32", name="prompt-b5-f32"),
        # one more continuation of a short sequence in a small model: one partly filled page of each layer
        _pages(1, 21, 4, 4, 64, fork=True, name="pages-fork-1"),
        # a prompt forked for sixty-three more samples, the headline's layers and heads
        _pages(63, 37, 24, 32, 64, fork=True, name="pages-fork-63"),
        # a cache of grouped heads moved into a new storage, page by page
        _pages(600, 64, 32, 8, 128, name="pages-move-600"),
        # the recurrent states and convolution rows of a forked sequence
        _slots(31, 4, 64 * 64 * 128, 3 * 4352, name="slots-fork-31"),
    ]


LAYOUTS = [(16, 4, 64, 64), (32, 32, 64, 64), (32, 8, 64, 64), (32, 8, 128, 128), (16, 4, 64, 128), (8, 1, 128, 128), (10, 2, 48, 48),
           (12, 3, 96, 96), (7, 7, 80, 80)]
MOST_PAIRS = 64 * 8500 * 32 * 256            # (row, key) pairs x heads x elements of a decode case
MOST_PAIRS_RUNS = 64 * 27 * 16384 * 32 * 256 // 2
MOST_PAIRS_F32 = 64 * 27 * 600 * 32 * 128


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.random()
    if kind < 0.15:
        fork = rng.random() < 0.6
        units, heads, dim, vdim = rng.choice([(4, 4, 64, 64), (24, 32, 64, 64), (16, 8, 64, 64), (32, 8, 128, 128), (6, 1, 576, 64), (3, 5, 36, 20)])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        size = units * heads * (dim + vdim) * 64 * (2 if dtype == "bfloat16" else 4)
        return _pages(_log(rng, 1, max(2, min(600, 2_400_000_000 // size))), rng.choice([0, 64, rng.randint(1, 63)]), units, heads, dim, vdim, fork, dtype)
    if kind < 0.25:
        return _slots(_log(rng, 1, 31), rng.randint(1, 6), rng.choice([7, 4096, 128 * 128 * 8, 64 * 64 * 128]), rng.choice([3 * 4352, 3 * 1281, 5]))
    heads, kv, dim, vdim = rng.choice(LAYOUTS)
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    runs = rng.random() < 0.4
    seqs = _log(rng, 1, 96 if not runs else 64)
    tokens = _log(rng, 2, 300) if runs else 1
    prefix = _log(rng, 20, 16384)
    private = rng.choice([0, 1, 63, 64, 65, _log(rng, 2, 1000)])
    most = MOST_PAIRS_F32 if dtype == "float32" else MOST_PAIRS_RUNS if runs else MOST_PAIRS
    groups = rng.choice([0, 0, 2, 3, 5])
    group_prefix = _log(rng, 10, 1500) if groups else 0
    while seqs * tokens * (prefix + private + group_prefix + tokens) * heads * (dim + vdim) > most:
        if tokens > 8:
            tokens //= 2
        elif prefix > 400:
            prefix = prefix * 2 // 3
        elif seqs > 1:
            seqs -= seqs // 3 + 1 if seqs > 2 else 1
        else:
            private, group_prefix = private // 2, group_prefix // 2
    return _attn(seqs, prefix, private, tokens, groups, group_prefix, heads, kv, dim, vdim, rng.choice([0.0, 0.0, 20.0]),
                 rng.random() < 0.3, dtype)


# --------------------------------------------------------------------------- what a case is made of
def _lengths(c):
    """(positions held before the step, new tokens) of every sequence."""
    out = []
    for i in range(c["seqs"]):
        held = c["prefix"] + (c["group_prefix"] if c["groups"] else 0) + ((i * 37 + 11) % (c["private"] + 1) if c["private"] else 0)
        new = 1 if c["tokens"] == 1 else 1 + (i * 29 + 7) % c["tokens"]
        out.append((held, new))
    return out


def _tables(c, seed):
    """Page ids [seqs, pages], shared ones in the same places, drawn without order; how many pages there are."""
    lens = _lengths(c)
    common = c["prefix"] // PAGE
    behind = (c["prefix"] + c["group_prefix"]) // PAGE if c["groups"] else common
    table = np.full((c["seqs"], max(-(-(h + n) // PAGE) for h, n in lens)), -1, dtype=np.int32)
    n = common
    table[:, :common] = np.arange(common)
    first = {}
    for i, (held, new) in enumerate(lens):
        key = i % c["groups"] if c["groups"] else 0
        if key not in first:
            first[key] = np.arange(n, n + behind - common)
            n += behind - common
        table[i, common:behind] = first[key]
        more = -(-(held + new) // PAGE) - behind
        table[i, behind:behind + more] = np.arange(n, n + more)
        n += more
    order = np.random.RandomState(seed % (1 << 31)).permutation(n).astype(np.int32)
    return np.where(table >= 0, order[table], -1).astype(np.int32), n


def _random(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32 if math.prod(shape) < 1 << 28 else dtype).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    c = case
    if c["op"] == "attention":
        dtype = DTYPES[c["dtype"]]
        lens = _lengths(c)
        table, n_pages = _tables(c, seed)
        rows = sum(n for _, n in lens)
        pos = np.concatenate([np.arange(h, h + n) for h, n in lens]).astype(np.int32)
        s = {"case": c, "lens": lens, "table": torch.from_numpy(table).to(DEVICE), "tok_pos": torch.from_numpy(pos).to(DEVICE),
             "q": (1.5 * _random(gen, (rows, c["heads"] * c["dim"]), torch.float32)).to(dtype),
             "k": _random(gen, (n_pages, c["kv"], PAGE, c["dim"]), dtype), "v": _random(gen, (n_pages, c["kv"], PAGE, c["vdim"]), dtype),
             "sink": _random(gen, (c["heads"],), torch.float32) if c["sink"] else None, "scale": c["dim"] ** -0.5}
        if own:       # one plan serves all layers of a step, and the decode steps behind it until the batch changes
            from scriptling_llm_lib_b200.cache import SharePlan
            from scriptling_llm_lib_b200.csrc.bindings import KernelSet
            s["kernels"] = KernelSet(dtype).shared
            s["plan"] = SharePlan.build(table, [h for h, _ in lens], [n for _, n in lens], c["heads"], c["kv"],
                                        s["kernels"].shape(c["dim"], c["vdim"]), DEVICE)
            s["err"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        return s
    if c["op"] == "pages":
        dtype = DTYPES[c["dtype"]]
        order = torch.from_numpy(np.random.RandomState(seed % (1 << 31)).permutation(c["pairs"] + 1).astype(np.int32))
        shape = (c["units"], c["pairs"] + 1, c["heads"], PAGE)
        k, v = _random(gen, (*shape, c["dim"]), dtype), _random(gen, (*shape, c["vdim"]), dtype)
        rows = torch.tensor([c["rows"] or 1 + (i * 23 + 5) % PAGE for i in range(c["pairs"])], dtype=torch.int32)
        s = {"case": c, "rows": rows.to(DEVICE), "from": [k, v]}
        if c["fork"]:
            s["src"], s["dst"], s["to"] = order[:1].repeat(c["pairs"]).to(DEVICE), order[1:].to(DEVICE), s["from"]
        else:
            s["src"], s["dst"] = order[1:].to(DEVICE), torch.arange(c["pairs"], dtype=torch.int32, device=DEVICE)
            s["to"] = [torch.zeros_like(k), torch.zeros_like(v)]
        if own:
            from scriptling_llm_lib_b200.csrc.bindings import PageKernels
            s["kernels"], s["err"] = PageKernels(), torch.zeros(1, dtype=torch.int32, device=DEVICE)
        return s
    n = c["pairs"] + 1
    order = torch.from_numpy(np.random.RandomState(seed % (1 << 31)).permutation(n).astype(np.int32)).to(DEVICE)
    held = [_random(gen, (n, w), t) for _ in range(c["units"]) for w, t in ((c["state"], torch.float32), (c["conv"], torch.bfloat16))]
    s = {"case": c, "from": held, "to": held, "src": order[:1].repeat(c["pairs"]), "dst": order[1:].clone()}
    if own:
        from scriptling_llm_lib_b200.csrc.bindings import PageKernels
        s["kernels"], s["err"] = PageKernels(), torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if c["op"] == "attention":
        return _attention_own(s, c) if own else _attention_plain(s, c)
    if c["op"] == "pages":
        if own:
            s["kernels"].copy_pages(list(zip(s["from"], s["to"])), s["src"], s["dst"], s["rows"], s["err"])
        else:
            src, dst = s["src"].long(), s["dst"].long()
            whole = torch.arange(PAGE, device=DEVICE) < s["rows"][:, None]
            for a, b in zip(s["from"], s["to"]):
                for u in range(a.shape[0]):
                    b[u, dst] = torch.where(whole[:, None, :, None], a[u, src], b[u, dst])
        return s["to"]
    if own:
        s["kernels"].copy_slots(list(zip(s["from"], s["to"])), s["src"], s["dst"], s["err"])
    else:
        src, dst = s["src"].long(), s["dst"].long()
        for a, b in zip(s["from"], s["to"]):
            b[dst] = a[src]
    return s["to"]


def _attention_own(s, c):
    q = s["q"]
    out = torch.empty((q.shape[0], c["heads"] * c["vdim"]), dtype=q.dtype, device=q.device)
    part = torch.empty((s["plan"].part_floats(c["vdim"]),), dtype=torch.float32, device=q.device)
    s["kernels"].attn(q, out, s["tok_pos"], s["table"], s["k"], s["v"], s["plan"], part, s["scale"], s["err"], softcap=c["cap"] or None,
                      sink=s["sink"])
    return out


def _attention_plain(s, c):
    """Sequence by sequence over its own pages, in 32 bits, rounded once at the end."""
    H, G, q = c["heads"], c["kv"], s["q"]
    out = torch.empty((q.shape[0], H * c["vdim"]), dtype=q.dtype, device=q.device)
    row = 0
    for b, (held, new) in enumerate(s["lens"]):
        m = held + new
        pages = s["table"][b, :-(-m // PAGE)].long()
        k = s["k"][pages].transpose(1, 2).reshape(-1, G, c["dim"])[:m].float()
        v = s["v"][pages].transpose(1, 2).reshape(-1, G, c["vdim"])[:m].float()
        qs = q[row:row + new].float().view(new, G, H // G, c["dim"])
        x = torch.einsum("ngrd,mgd->grnm", qs, k) * s["scale"]
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        hidden = torch.arange(m, device=q.device)[None, :] > torch.arange(held, m, device=q.device)[:, None]
        x = x.masked_fill(hidden, -math.inf)
        top = x.amax(-1, keepdim=True)
        if s["sink"] is not None:
            z = s["sink"].view(G, H // G, 1, 1)
            top = torch.maximum(top, z)
        p = torch.exp(x - top)
        den = p.sum(-1, keepdim=True)
        if s["sink"] is not None:
            den = den + torch.exp(z - top)
        o = torch.einsum("grnm,mgd->ngrd", p, v) / den.permute(2, 0, 1, 3)
        out[row:row + new] = o.reshape(new, H * c["vdim"]).to(q.dtype)
        row += new
    return out


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    width = 2 if c.get("dtype") == "bfloat16" else 4
    if c["op"] == "attention":
        lens = _lengths(c)
        table, n_pages = _tables(c, 0)
        ends = {}                                            # positions in use of every page: what is read of it
        for row, (h, n) in zip(table, lens):
            for i in range(-(-(h + n) // PAGE)):
                ends[int(row[i])] = min(PAGE, h + n - i * PAGE)
        rows = sum(n for _, n in lens)
        pairs = sum(n * h + n * (n + 1) // 2 for h, n in lens)
        return {"bytes": width * (sum(ends.values()) * c["kv"] * (c["dim"] + c["vdim"]) + rows * c["heads"] * (c["dim"] + c["vdim"])),
                "flops": 2 * pairs * c["heads"] * (c["dim"] + c["vdim"])}
    if c["op"] == "pages":
        rows = [c["rows"] or 1 + (i * 23 + 5) % PAGE for i in range(c["pairs"])]
        read = max(rows) if c["fork"] else sum(rows)
        return {"bytes": width * c["units"] * c["heads"] * (c["dim"] + c["vdim"]) * (read + sum(rows)), "flops": 0}
    return {"bytes": c["units"] * (4 * c["state"] + 2 * c["conv"]) * (1 + c["pairs"]), "flops": 0}


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """Attention head by head from the definition. What copies give is no computed number."""
    c = case
    if c["op"] != "attention":
        return None
    s = prepare(case, seed)
    rep = c["heads"] // c["kv"]
    table = s["table"].cpu().numpy()
    out, first = [], 0
    for b, (held, new) in enumerate(s["lens"]):
        keys = np.arange(held + new)
        page, place = torch.from_numpy(table[b][keys // PAGE]).long().to(DEVICE), torch.from_numpy(keys % PAGE).to(DEVICE)
        q = s["q"][first:first + new].double().reshape(new, c["heads"], c["dim"])
        late = torch.from_numpy(keys).to(DEVICE) > s["tok_pos"][first:first + new, None]
        o = torch.empty((new, c["heads"], c["vdim"]), dtype=torch.float64, device=DEVICE)
        for g in range(c["kv"]):
            k, v = s["k"][page, g, place].double(), s["v"][page, g, place].double()
            for h in range(g * rep, (g + 1) * rep):
                score = q[:, h] @ k.T * s["scale"]
                if c["cap"]:
                    score = c["cap"] * torch.tanh(score / c["cap"])
                score[late] = -math.inf
                if s["sink"] is not None:
                    score = torch.cat([score, s["sink"][h].double().expand(new, 1)], 1)
                weight = torch.softmax(score, -1)
                o[:, h] = weight[:, :len(keys)] @ v
        out.append(o.reshape(new, -1))
        first += new
    return torch.cat(out)
