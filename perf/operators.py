"""Timed cases of two attention operators beside the paged layer attention, each one pass of a layer.

``shared``  attention of a step whose sequences share long prefixes in the paged cache (a system
            prompt, one document under many questions, several samples of one prompt): the step's
            K/V rows are stored to their pages, then every query attends over its sequence's
            keys, causally.  Sequences come in groups written ``sequences x prefix tokens``; each
            has tokens of its own after the prefix (``clo``..``chi`` cached, ``nlo``..``nhi`` new).
``cross``   attention of each sequence's queries over all keys of an encoder's states of another
            length, held in a pool of rows.  ``beams`` sequences in a row read one request's
            states; ``full`` is the encoder's own layer (queries and keys of one sequence, each
            seen by each).

Head shapes are those of the model families the library serves, and generic encoder shapes.  A
case's lengths come from ``layout``; the inputs, and the order of pages and rows, from the seed.
"""

import functools
import math
import os
import sys

import numpy as np
import torch

own = False  # the framework's operators; False: their plain form in elementary operations

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# q heads, KV heads, head dim.
SHAPES = {
    "16/8/128": (16, 8, 128),
    "32/8/128": (32, 8, 128),
    "40/8/128": (40, 8, 128),
    "32/8/64": (32, 8, 64),
    "4/1/256": (4, 1, 256),
    "8/1/512": (8, 1, 512),
    "12/12/64": (12, 12, 64),
    "16/16/64": (16, 16, 64),
}


def _shared(name, shape, groups, *, clo, chi, nlo=1, nhi=1, block=256, layout=0):
    case = dict(kind="shared", shape=shape, groups=groups, clo=clo, chi=chi, nlo=nlo, nhi=nhi,
                block=block, layout=layout)
    if name:
        case["name"] = name
    return case


def _cross(name, shape, requests, *, klo, khi, beams=1, qlo=1, qhi=1, full=False, packed=True,
           layout=0):
    case = dict(kind="cross", shape=shape, requests=requests, beams=beams, klo=klo, khi=khi,
                qlo=qlo, qhi=qhi, full=full, packed=packed, layout=layout)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # A few samples of one short prompt: launches and latency count.
        _shared("shared_decode_6_samples", "16/8/128", "6x512", clo=1, chi=90),
        # A chat service with one long system prompt, a full decode batch.
        _shared("shared_decode_64_rows", "32/8/128", "64x8192", clo=16, chi=1500),
        # Several documents under question at once, and rows that share nothing.
        _shared("shared_decode_4_groups", "16/8/128", "97x8192,61x4096,57x2048,41x0", clo=40,
                chi=2000),
        # Multi-query heads over small pages.
        _shared("shared_decode_mqa_d256", "4/1/256", "33x6144", clo=1, chi=700, block=16),
        # d = 64 and a medium batch under a very long document.
        _shared("shared_decode_20_rows_d64", "32/8/64", "20x24576", clo=1, chi=400),
        # Questions arriving together on one cached document: odd lengths, one-token ones too.
        _shared("shared_prefill_questions", "32/8/128", "24x8192", clo=0, chi=0, nlo=1, nhi=160),
        # Single tokens of a few sequences over short encoder states, one of them empty.
        _cross("cross_decode_5_rows", "16/16/64", 5, klo=0, khi=700),
        # A full decode batch over encoder states of up to 1500 rows, as a packed kv projection.
        _cross("cross_decode_128_rows", "16/16/64", 128, klo=300, khi=1500),
        # Beam search: five beams of each request read the same states.
        _cross("cross_decode_40x5_beams", "32/8/128", 40, beams=5, klo=500, khi=4000,
               packed=False),
        # A text encoder's layer over a batch of short passages.
        _cross("cross_full_48_passages", "12/12/64", 48, klo=9, khi=512, full=True),
        # A decoder's prompts over long encoder states.
        _cross("cross_prefill_long", "32/8/128", 6, klo=2000, khi=9000, qlo=130, qhi=900),
        # Prompts of a multi-query decoder with wide heads over medium states.
        _cross("cross_prefill_mqa_d256", "4/1/256", 9, klo=100, khi=3000, qlo=2, qhi=500,
               packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; no larger than the largest listed one."""
    while True:
        case = _draw(rng)
        w = work(case)
        rows, width = _padded_size(case)
        if 0 < w["bytes"] <= 1.5e9 and w["flops"] <= 2.5e11 and rows * width * 8 <= 22e9:
            return case


def _draw(rng):
    layout = rng.randrange(1 << 20)
    if rng.random() < 0.5:
        shape = rng.choice([s for s in sorted(SHAPES) if s != "12/12/64"])
        block = rng.choice([256, 256, 64, 16])
        groups, left = [], _log(rng, 2, 200)
        while left > 0 and len(groups) < 5:
            n = min(left, _log(rng, 1, 128))
            prefix = 0 if rng.random() < 0.15 else block * max(1, _log(rng, 64, 24000) // block)
            groups.append(f"{n}x{prefix}")
            left -= n
        chi = _log(rng, 1, 3000)
        nhi = 1 if rng.random() < 0.6 else _log(rng, 2, 400)
        return _shared(None, shape, ",".join(groups), clo=rng.choice([0, chi // 8]), chi=chi,
                       nlo=1, nhi=nhi, block=block, layout=layout)
    shape = rng.choice(sorted(SHAPES))
    full = rng.random() < 0.25
    khi = _log(rng, 1, 2000 if full else 9000)
    klo = rng.choice([0, 1, khi // 8, khi])
    beams = 1 if full else rng.choice([1, 1, 2, 4, 7])
    qhi = rng.choice([1, _log(rng, 1, 900)])
    return _cross(None, shape, _log(rng, 1, 128), klo=klo, khi=khi, beams=beams,
                  qlo=rng.choice([1, qhi]), qhi=qhi, full=full, packed=rng.random() < 0.5,
                  layout=layout)


@functools.lru_cache(maxsize=64)
def _sequences(groups, clo, chi, nlo, nhi, layout):
    """(group, prefix, own cached, new) of every sequence of a shared step."""
    r = np.random.default_rng(layout)
    got = []
    for g, part in enumerate(groups.split(",")):
        n, prefix = (int(x) for x in part.split("x"))
        got += [(g, prefix, int(r.integers(clo, chi + 1)), int(r.integers(nlo, nhi + 1)))
                for _ in range(n)]
    return tuple(got)


def _seqs(case):
    return _sequences(*(case[k] for k in ("groups", "clo", "chi", "nlo", "nhi", "layout")))


@functools.lru_cache(maxsize=64)
def _requests(requests, beams, klo, khi, qlo, qhi, full, layout):
    """(request, queries, keys) of every sequence of a cross step."""
    r = np.random.default_rng(layout)
    keys = [int(x) for x in r.integers(klo, khi + 1, requests)]
    return tuple((i, k if full else int(r.integers(qlo, qhi + 1)), k)
                 for i, k in enumerate(keys) for _ in range(beams))


def _reqs(case):
    return _requests(*(case[k] for k in ("requests", "beams", "klo", "khi", "qlo", "qhi", "full",
                                         "layout")))


def _lengths(case):
    """(queries, keys) of every sequence."""
    if case["kind"] == "cross":
        return [(n, k) for _, n, k in _reqs(case)]
    return [(n, p + c + n) for _, p, c, n in _seqs(case)]


def _padded_size(case):
    """Sequences x longest keys, and K values of one key: what the plain form lays out."""
    _, hkv, d = SHAPES[case["shape"]]
    both = _lengths(case)
    return len(both) * max(1, max(k for _, k in both)), hkv * d


def _scale(case):
    return float(np.float32(SHAPES[case["shape"]][2] ** -0.5))


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + salt)
    return g


def _fill(flat, seed, salt):
    g = _gen(seed, salt)
    for s in range(0, flat.numel(), 1 << 28):
        flat[s:s + (1 << 28)].normal_(generator=g)


def _places(case, seed):
    """Where each sequence's keys are: slots of the arena's pages (shared; with the block tables
    and the number of blocks) or rows of the encoder pool (cross; with the pool's size)."""
    r = np.random.default_rng(seed)
    if case["kind"] == "cross":
        reqs = _reqs(case)
        keys = {i: k for i, _, k in reqs}
        start, at = {}, int(r.integers(0, 8))
        for i in r.permutation(len(keys)):
            start[int(i)] = at
            at += keys[int(i)] + int(r.integers(0, 8))
        return [np.arange(start[i], start[i] + k) for i, _, k in reqs], None, max(1, at)
    bs, seqs = case["block"], _seqs(case)
    shared = {g: p // bs for g, p, _, _ in seqs}
    own_pages = [-(-(p + c + n) // bs) - p // bs for _, p, c, n in seqs]
    total = sum(shared.values()) + sum(own_pages)
    blocks = total + max(1, total // 10)
    ids = iter(r.permutation(blocks)[:total].tolist())
    heads = {g: [next(ids) for _ in range(m)] for g, m in shared.items()}
    tables = [heads[g] + [next(ids) for _ in range(m)] for (g, _, _, _), m in zip(seqs, own_pages)]
    slots = [(np.asarray(t, np.int64)[:, None] * bs + np.arange(bs)).reshape(-1)[:p + c + n]
             for t, (_, p, c, n) in zip(tables, seqs)]
    return slots, tables, blocks


def _inputs(case, seed, tokens):
    """q, and for a shared step the new k and v rows."""
    hq, hkv, d = SHAPES[case["shape"]]
    q = torch.randn(tokens, hq, d, device="cuda", generator=_gen(seed, 1))
    if case["kind"] == "cross":
        return q, None, None
    return (q, *(torch.randn(tokens, hkv, d, device="cuda", generator=_gen(seed, s)) for s in (2, 3)))


def _pool(case, seed, rows):
    """The encoder's keys and values: views of one packed projection, or two tensors."""
    _, hkv, d = SHAPES[case["shape"]]
    kv = torch.empty((rows, 2, hkv, d) if case["packed"] else (2, rows, hkv, d), device="cuda")
    _fill(kv.view(-1), seed, 4)
    return kv.unbind(1 if case["packed"] else 0)


class _Memory:
    """Device memory of the arena as torch.as_tensor takes it; keeps its owner alive."""

    def __init__(self, ptr, count, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": (count,), "typestr": "<f4",
                                         "data": (ptr, False), "version": 2, "strides": None}


class _Engine:
    """What an engine keeps over its steps, and the step it has set on its context."""

    def __init__(self, case, tables, blocks, places):
        pkg = os.path.join(_ROOT, "nano-vllm-java_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import nanollvm_amd as nva
        from nanollvm_amd import step

        hq, hkv, d = SHAPES[case["shape"]]
        both = _lengths(case)
        decode = all(n == 1 for n, _ in both) and not case.get("full")
        lens = np.asarray([k for _, k in both], np.int32)
        cu_q = np.concatenate([[0], np.cumsum([n for n, _ in both])]).astype(np.int32)
        cu_k = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.arena = None
        self.ctx = nva.Context(0)
        when = (dict(is_prefill=False, context_lens=lens) if decode else
                dict(is_prefill=True, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k,
                     max_seqlen_q=max(n for n, _ in both), max_seqlen_k=int(lens.max())))
        if case["kind"] == "cross":
            self.ctx.set(**when)
            self.ctx.set_encoder([int(p[0]) if len(p) else 0 for p in places], lens)
            self.layer = nva.CrossAttention(hq, d, _scale(case), hkv)
            return
        self.arena = nva.KvCacheArena(self.ctx, 1, blocks, case["block"], hkv, d)
        width = max(len(t) for t in tables)
        table = np.full((len(tables), width), -1, np.int32)
        for i, t in enumerate(tables):
            table[i, :len(t)] = t
        new = np.concatenate([p[len(p) - n:] for p, (n, _) in zip(places, both)])
        self.ctx.set(slot_mapping=new, block_tables=table, **when)
        self.ctx.share_prefixes(step.find_shared_prefixes(
            table, [k - n for n, k in both], case["block"]))
        self.ctx.bind_kv_cache(self.arena)
        self.layer = nva.Attention(hq, d, _scale(case), hkv)

    def pages(self):
        k, v, nbytes = self.arena.device_ptrs(0)
        return [torch.as_tensor(_Memory(p, nbytes // 4, self), device="cuda") for p in (k, v)]

    def forward(self, q, k, v):
        return self.layer.forward(q, k, v, self.ctx)

    def __del__(self):
        for x in (getattr(self, "arena", None), getattr(self, "ctx", None)):
            if x is not None:
                x.close()


def prepare(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    places, tables, size = _places(case, seed)
    both = _lengths(case)
    tokens = sum(n for n, _ in both)
    s = {"kind": case["kind"], "scale": _scale(case)}
    s["q"], s["k_new"], s["v_new"] = _inputs(case, seed, tokens)
    if own:
        s["engine"] = _Engine(case, tables, size, places)
    else:
        s.update(_padded(both, places, case["kind"] == "shared"))
    if case["kind"] == "cross":
        s["k"], s["v"] = _pool(case, seed, size)
    else:
        count = size * case["block"] * hkv * d
        s["k"], s["v"] = ([x.view(-1, hkv, d) for x in s["engine"].pages()] if own else
                          [torch.empty(count, device="cuda").view(-1, hkv, d) for _ in range(2)])
        for x, salt in ((s["k"], 4), (s["v"], 5)):
            _fill(x.view(-1), seed, salt)
    return s


def _padded(both, places, causal):
    """The plain form's plan: each sequence's key rows and query rows, padded to the longest, how
    many keys each query sees, where each row of the output is, and the new rows' places."""
    nq, nk = max(1, max(n for n, _ in both)), max(1, max(k for _, k in both))
    keys = np.zeros((len(both), nk), np.int64)
    rows = np.zeros((len(both), nq), np.int64)
    seen = np.zeros((len(both), nq), np.int64)
    at, back, new = 0, [], []
    for b, ((n, k), p) in enumerate(zip(both, places)):
        keys[b, :k] = p
        rows[b, :n] = np.arange(at, at + n)
        seen[b, :n] = np.arange(k - n + 1, k + 1) if causal else k
        back.append(b * nq + np.arange(n))
        new.append(p[k - n:] if causal else [])
        at += n
    dev = [torch.from_numpy(np.asarray(x, np.int64)).cuda()
           for x in (keys, rows, seen, np.concatenate(back), np.concatenate(new))]
    return dict(zip(("keys", "rows", "seen", "back", "new"), dev))


def _plain(s):
    """softmax(scale q k^T) v of every sequence as one padded batch."""
    q, k, v = s["q"][s["rows"]], s["k"][s["keys"]], s["v"][s["keys"]]
    n, nq, hq, d = q.shape
    nk, hkv = k.shape[1:3]
    rep = hq // hkv
    q = q.view(n, nq, hkv, rep, d).permute(0, 2, 1, 3, 4).reshape(n * hkv, nq * rep, d)
    k = k.permute(0, 2, 3, 1).reshape(n * hkv, d, nk).contiguous()
    x = torch.bmm(q, k).mul_(s["scale"]).view(n, hkv, nq, rep, nk)
    del q, k
    unseen = torch.arange(nk, device=x.device) >= s["seen"][:, None, :, None, None]
    x.masked_fill_(unseen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = v.permute(0, 2, 1, 3).reshape(n * hkv, nk, d).contiguous()
    o = torch.bmm(x.view(n * hkv, nq * rep, nk), v).view(n, hkv, nq, rep, d)
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    return o.permute(0, 2, 1, 3, 4).reshape(n * nq, hq, d)[s["back"]]


def run(state):
    s = state
    if s["kind"] == "cross":
        return {"out": s["engine"].forward(s["q"], s["k"], s["v"]) if own else _plain(s)}
    if own:
        out = s["engine"].forward(s["q"], s["k_new"], s["v_new"])
    else:
        s["k"][s["new"]] = s["k_new"]
        s["v"][s["new"]] = s["v_new"]
        out = _plain(s)
    return {"out": out, "k": s["k"], "v": s["v"]}


def work(case):
    hq, hkv, d = SHAPES[case["shape"]]
    both = _lengths(case)
    tokens = sum(n for n, _ in both)
    if case["kind"] == "cross":
        keys = sum({i: k for i, _, k in _reqs(case)}.values())
        pairs = sum(n * k for n, k in both)
        moved = 2 * tokens * hq * d + 2 * keys * hkv * d
    else:  # q read, out written, the new rows read and written, the cached rows read once
        seqs = _seqs(case)
        keys = sum({g: p for g, p, _, _ in seqs}.values()) + sum(c for _, _, c, _ in seqs)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in both)
        moved = 2 * tokens * hq * d + (4 * tokens + 2 * keys) * hkv * d
    return {"bytes": 4.0 * moved, "flops": 4.0 * d * hq * pairs}


def exact(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    rep, scale, causal = hq // hkv, _scale(case), case["kind"] == "shared"
    places, _, size = _places(case, seed)
    both = _lengths(case)
    q, k_new, v_new = _inputs(case, seed, sum(n for n, _ in both))
    if causal:
        k, v = (torch.empty(size * case["block"], hkv, d, device="cuda") for _ in range(2))
        _fill(k.view(-1), seed, 4)
        _fill(v.view(-1), seed, 5)
    else:
        k, v = _pool(case, seed, size)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for (n, keys), p in zip(both, places):  # the new rows first: later sequences read none of them
        if causal:
            t = torch.from_numpy(p[keys - n:]).cuda()
            k[t], v[t] = k_new[at:at + n], v_new[at:at + n]
        if n and keys:
            rows = torch.from_numpy(p).cuda()
            kk, vv = k[rows].double(), v[rows].double()
            for h in range(hkv):
                heads = q[at:at + n, h * rep:(h + 1) * rep].double().reshape(n * rep, d)
                logits = (heads @ kk[:, h].T.contiguous()).view(n, rep, keys) * scale
                if causal:
                    ahead = torch.ones(n, keys, dtype=torch.bool, device="cuda").triu(keys - n + 1)
                    logits = logits.masked_fill(ahead[:, None], -math.inf)
                weights = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp()
                out[at:at + n, h * rep:(h + 1) * rep] = \
                    (weights.view(n * rep, keys) @ vv[:, h].contiguous()).view(n, rep, d)
        at += n
    return {"out": out, "k": k.double(), "v": v.double()} if causal else {"out": out}
