"""Timed operators of a server that keeps many sequences in one pool of cache pages.

Four operators make one round of such a server: a prompt's keys and values move between the dense planes that prefill
works on and the pages of a sequence (``copy``), one new token of every sequence attends to the pages it owns
(``attention``), a sequence that has grown too long gives up the rows that drew the least attention (``evict``), and the
next token is chosen from logits after penalties, biases and a grammar's mask (``choose``).

Every function below has two forms.  Where ``own`` is false it computes the operator from elementary torch operations;
where it is true it makes the calls of the operator ABI.  Both work on the same storage: tensors that, in the second
form, lie in the library's buffers.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_NONE = -1  # a page id, a length or a token that is none: 0xffffffff as a signed word


# ---- cases ----------------------------------------------------------------------------------------


def _attention(name, seqs, longest, heads, kv_heads, head_dim, page, window=0, weights=False, dropped=0):
    return {"name": name, "kind": "attention", "seqs": seqs, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "n_rot": head_dim, "page": page, "window": window, "weights": weights, "dropped": dropped}


def _evict(name, seqs, longest, kv_heads, head_dim, page, keep, first, recent):
    return {"name": name, "kind": "evict", "seqs": seqs, "longest": longest, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "keep": keep, "first": first, "recent": recent}


def _copy(name, seqs, longest, kv_heads, head_dim, page, to_pages):
    return {"name": name, "kind": "copy", "seqs": seqs, "longest": longest, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "to_pages": to_pages}


def _choose(name, rows, vocab, history, biases, mask):
    return {"name": name, "kind": "choose", "rows": rows, "vocab": vocab, "history": history, "biases": biases, "mask": mask}


def listed():
    return [
        # The second token of a short chat turn: one sequence, two pages, all latency.
        _attention("attend 1 x 17", 1, 17, 16, 8, 128, 16),
        # A server's batch in mid-answer, ragged.
        _attention("attend 32 x 1000", 32, 1000, 16, 8, 128, 64),
        # The wider decoder's batch, caches evicted before and counted again for the next time.
        _attention("attend 32 x 4095 weights", 32, 4095, 32, 8, 128, 64, weights=True, dropped=1500),
        # One request over a book: the cache's length is all the parallelism there is.
        _attention("attend 1 x 131071", 1, 131071, 32, 8, 128, 128),
        # Sliding-window layers with one KV head of 256: the pages before the window are gone.
        _attention("attend 8 x 5000 window", 8, 5000, 4, 1, 256, 16, window=512),
        # One long conversation is cut down to a small cache, odd sizes.
        _evict("evict 1 x 1001", 1, 1001, 8, 128, 16, 300, 4, 33),
        # A batch is halved.
        _evict("evict 32 x 4096", 32, 4096, 8, 128, 64, 2048, 4, 256),
        # A prompt that has just been prefilled goes into its pages.
        _copy("copy 1 x 300", 1, 300, 8, 128, 16, True),
        # Paged prompts come back to the dense planes for their next chunk.
        _copy("copy 16 x 2048 back", 16, 2048, 8, 128, 64, False),
        # One request with penalties only.
        _choose("choose 1 of 151936", 1, 151936, 600, 0, False),
        # A batch under grammars, with long histories and a bias map each.
        _choose("choose 32 of 151936 masked", 32, 151936, 4000, 300, True),
        # The largest head and a wide batch.
        _choose("choose 48 of 262144", 48, 262144, 1200, 16, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    kind = rng.choice(["attention", "attention", "evict", "copy", "choose"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads, head_dim = rng.choice([(8, 128), (8, 128), (4, 128), (1, 256), (2, 64), (4, 32)])
    if kind == "attention":
        c = _attention("", _log_int(rng, 1, 64), _log_int(rng, 1, 130000), kv_heads * rng.choice([1, 2, 4, 5, 8]), kv_heads,
                       head_dim, page, rng.choice([0, 0, 0, _log_int(rng, 1, 4000)]), rng.random() < 0.4,
                       rng.choice([0, 0, _log_int(rng, 1, 30000)]))
        c["n_rot"] = rng.choice([head_dim, head_dim, head_dim // 2])
    elif kind == "evict":
        longest = _log_int(rng, 2, 16000)
        keep = rng.randint(1, longest)
        first = rng.randint(0, min(keep, 8))
        c = _evict("", _log_int(rng, 1, 48), longest, kv_heads, head_dim, page, keep, first, rng.randint(0, (keep - first) // 2))
    elif kind == "copy":
        c = _copy("", _log_int(rng, 1, 48), _log_int(rng, 1, 8000), kv_heads, head_dim, page, rng.random() < 0.5)
    else:
        c = _choose("", _log_int(rng, 1, 64), rng.choice([512, 32001, 151936, 262144]), _log_int(rng, 1, 8000),
                    rng.choice([0, _log_int(rng, 1, 1000)]), rng.random() < 0.5)
    del c["name"]
    return c


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), _cost(work(c)))
    while True:
        case = _draw_one(rng)
        if _cost(work({**case, "window": 0})) <= most[case["kind"]]:  # the cache is held whole, whatever a window sees of it
            return case


def _cost(w):
    return max(w["bytes"], w["flops"] / 200)


def _lengths(case):
    """Ragged lengths, from a quarter of the longest to the longest."""
    n = case["longest"]
    return [max(1, n - int(0.75 * n * ((s * 0.6180339887) % 1.0))) for s in range(case["seqs"])]


def work(case):
    kind = case["kind"]
    if kind == "choose":
        rows, n = case["rows"], case["vocab"]
        nbytes = 8.0 * rows * n + rows * (4.0 * case["history"] + 8.0 * case["biases"] + 20)
        return {"bytes": nbytes + (rows * n / 8.0 if case["mask"] else 0), "flops": float(rows * n)}
    lens = _lengths(case)
    row = 4.0 * case["kv_heads"] * case["head_dim"]  # a position's key and value in f16, all heads
    if kind == "copy":
        return {"bytes": 2 * row * sum(lens), "flops": 0.0}
    if kind == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": 2 * row * kept + 4.0 * case["kv_heads"] * (sum(lens) + 2 * kept), "flops": 0.0}
    seen = sum(min(n + 1, case["window"] or n + 1) for n in lens)  # the new token sees itself
    heads, hd, s = case["heads"], case["head_dim"], case["seqs"]
    nbytes = row * seen + 4.0 * s * hd * (2 * heads + 2 * case["kv_heads"]) + 4.0 * seen / case["page"]
    if case["weights"]:
        nbytes += 8.0 * case["kv_heads"] * seen
    return {"bytes": nbytes, "flops": 4.0 * heads * hd * seen}


# ---- inputs ---------------------------------------------------------------------------------------

_CONTEXT = []


def _context():
    from tuckmill_b200 import cuda
    if not _CONTEXT:
        _CONTEXT.append(cuda.CudaContext(0))
    return _CONTEXT[0]


class _DeviceArray:
    """A library buffer as torch sees it: bytes."""

    def __init__(self, buf):
        self.__cuda_array_interface__ = {"shape": (len(buf),), "typestr": "|u1", "data": (buf.device_ptr(), False), "version": 3}


class _Storage:
    """A buffer of the library's.  A program keeps its caches, tables and workspaces and fills them again: so a buffer that
    no state and no result holds any more serves the next state of its case, as torch does with the storage of its tensors.
    Every tensor in it is filled anew; a workspace needs no filling."""

    _spare, _used, _of = {}, False, None  # by size; whether one was in use since the last wait; of which case

    def __init__(self, nbytes):
        self.b = _context().buffer(nbytes)
        self.bytes, self.all = nbytes, torch.as_tensor(_DeviceArray(self.b), device=_DEV)

    @classmethod
    def take(cls, nbytes):
        spare = cls._spare.get(nbytes)
        if not spare:
            return _Lease(cls(nbytes))
        if cls._used:
            torch.cuda.synchronize()  # what used the spare buffers has ended
            cls._used = False
        return _Lease(spare.pop())

    @classmethod
    def give(cls, storage):
        cls._used = True
        cls._spare.setdefault(storage.bytes, []).append(storage)

    @classmethod
    def keep_only(cls, case):
        if cls._of != case:
            cls._spare.clear()
            cls._of = dict(case)


class _Lease:
    """Held by whoever uses a storage: a tensor in it, or a state whose workspace it is."""

    def __init__(self, storage):
        self.storage, self.b = storage, storage.b

    def tensor(self, like):
        t = self.storage.all.view(like.dtype).view(like.shape)
        t.lease = self
        return t

    def __del__(self):
        _Storage.give(self.storage)


class _Held:
    """A tensor, and the library's buffer that it lies in where a caller of the library made it."""

    def __init__(self, t):
        self.t, self.b = t, None
        if own:
            lease = _Storage.take(t.numel() * t.element_size())
            self.b, self.t = lease.b, lease.tensor(t)
            self.t.copy_(t)


def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    return g


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _pages_of(case, lens, sets=1):
    """Tables [sets][seqs][max_pages] that name every page once, in no order, and the number of pages."""
    page = case["page"]
    max_pages = -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    return max_pages, need, sets * sum(need) + 3


def _tables(g, max_pages, need, pages, sets=1):
    order = torch.randperm(pages, device=_DEV, generator=g).to(torch.int32)
    slot = torch.arange(max_pages, device=_DEV)
    n = _words(need).long()
    start = torch.cumsum(n, 0) - n
    out = []
    for i in range(sets):
        at = (start[:, None] + slot[None, :] + i * int(sum(need))).clamp(max=pages - 1)
        out.append(torch.where(slot[None, :] < n[:, None], order[at], torch.full_like(order[at], _NONE)))
    return out


def _pool(g, case, pages):
    return torch.randn(pages, case["kv_heads"], case["page"], case["head_dim"], dtype=torch.float16, device=_DEV, generator=g)


def prepare(case, seed):
    g = _gen(seed)
    state = {"attention": _prepare_attention, "evict": _prepare_evict, "copy": _prepare_copy,
             "choose": _prepare_choose}[case["kind"]](case, g)
    state["case"] = case
    if own:
        state["ctx"] = _context()
        _Storage.keep_only(case)
        torch.cuda.synchronize()  # what torch wrote is complete before the library's stream reads it
    return state


def _prepare_attention(case, g):
    s, heads, kvh, hd = case["seqs"], case["heads"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    max_pages, need, pages = _pages_of(case, [n + 1 for n in lens])
    (table,) = _tables(g, max_pages, need, pages)
    if case["window"]:  # pages wholly before the window are given back
        gone = torch.clamp(_words(lens) + 1 - case["window"], min=0) // case["page"]
        table = torch.where(torch.arange(max_pages, device=_DEV)[None, :] < gone[:, None], torch.full_like(table, _NONE), table)
    st = {
        "qkv": _Held(torch.randn(s, (heads + 2 * kvh) * hd, device=_DEV, generator=g)),
        "q_norm": _Held(1 + 0.1 * torch.randn(hd, device=_DEV, generator=g)),
        "k_norm": _Held(1 + 0.1 * torch.randn(hd, device=_DEV, generator=g)),
        "inv_freq": _Held(_inv_freq(case["n_rot"])),
        "k": _Held(_pool(g, case, pages)), "v": _Held(_pool(g, case, pages)),
        "table": _Held(table), "lens": _Held(_words(lens)), "pos": _Held(_words([n + case["dropped"] for n in lens])),
        "out": _Held(torch.zeros(s, heads * hd, device=_DEV)), "status": _Held(_words([0])),
        "max_pages": max_pages, "pages": pages,
    }
    if case["weights"]:  # what earlier tokens gave to each cached row
        before = torch.rand(s, kvh, max_pages * case["page"], device=_DEV, generator=g).pow(4)
        st["weights"], st["weights_out"] = _Held(before), _Held(torch.zeros_like(before))
    if own:
        from tuckmill_b200 import cuda
        n = st["qkv"].b.len()
        off = [0, heads * hd * 4, (heads + kvh) * hd * 4]
        st["views"] = [st["qkv"].b.view(o, n - o) for o in off]
        st["scratch"] = _Storage.take(cuda.attention_paged_scratch_bytes(s, heads, kvh, hd, case["page"], max_pages,
                                                                      case["weights"]))
    return st


def _inv_freq(n_rot):
    """Rotation frequencies of base 1e6, rounded to f32 once."""
    f = 1e6 ** (-np.arange(n_rot // 2, dtype=np.float64) * 2 / n_rot)
    return torch.from_numpy(f.astype(np.float32)).to(_DEV)


def _prepare_evict(case, g):
    s, kvh, keep = case["seqs"], case["kv_heads"], case["keep"]
    lens = _lengths(case)
    max_pages, need, pages = _pages_of(case, lens, 2)
    table, to = _tables(g, max_pages, need, pages, 2)
    cap = max_pages * case["page"]
    weights = torch.rand(s, kvh, cap, device=_DEV, generator=g).pow(8)  # a few rows draw most of the attention
    weights = torch.where(weights < 1e-6, torch.zeros_like(weights), weights)  # rows never looked at tie
    return {"k": _Held(_pool(g, case, pages)), "v": _Held(_pool(g, case, pages)), "table": _Held(table), "to": _Held(to),
            "lens": _Held(_words(lens)), "lens_out": _Held(_words([0] * s)), "weights": _Held(weights),
            "weights_out": _Held(torch.zeros_like(weights)), "status": _Held(_words([0])),
            "kept": _Held(torch.zeros(s, kvh, keep, dtype=torch.int32, device=_DEV)), "max_pages": max_pages, "pages": pages}


def _prepare_copy(case, g):
    s, kvh, hd = case["seqs"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    max_pages, need, pages = _pages_of(case, lens)
    (table,) = _tables(g, max_pages, need, pages)
    cap = max(lens)
    # every other sequence carries on from a third of its length
    runs = [(i, i, n // 3 if i % 2 else 0, n - (n // 3 if i % 2 else 0)) for i, n in enumerate(lens)]
    dense = lambda: torch.randn(s, kvh, cap, hd, dtype=torch.float16, device=_DEV, generator=g)  # noqa: E731
    return {"k": _Held(_pool(g, case, pages)), "v": _Held(_pool(g, case, pages)), "kc": _Held(dense()), "vc": _Held(dense()),
            "table": _Held(table), "status": _Held(_words([0])), "runs": runs, "runs_dev": _words(runs).long(),
            "rows": sum(r[3] for r in runs), "cap": cap, "max_pages": max_pages, "pages": pages}


def _prepare_choose(case, g):
    r, n, h, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    hist = [max(1, h - int(0.75 * h * ((i * 0.6180339887) % 1.0))) for i in range(r)]
    stride = h + 8
    # text repeats itself: half of the tokens come from a few hundred
    common = torch.randint(0, n, (r, 200), device=_DEV, generator=g)
    pick = torch.randint(0, 200, (r, stride), device=_DEV, generator=g)
    rare = torch.randint(0, n, (r, stride), device=_DEV, generator=g)
    half = torch.rand(r, stride, device=_DEV, generator=g) < 0.5
    log = torch.where(half, torch.gather(common, 1, pick), rare).to(torch.int32)
    pen = torch.stack([1 + 0.3 * torch.rand(r, device=_DEV, generator=g), 0.5 * torch.rand(r, device=_DEV, generator=g),
                       0.2 * torch.rand(r, device=_DEV, generator=g)], 1)
    st = {"x": _Held(4 * torch.randn(r, n, device=_DEV, generator=g)), "y": _Held(torch.zeros(r, n, device=_DEV)),
          "log": _Held(log), "pos": _Held(_words([v - 1 for v in hist])), "prompt": _Held(_words([v // 2 for v in hist])),
          "pen": _Held(pen.contiguous()), "stride": stride}
    if nb:
        st["bias_ids"] = _Held(torch.randint(0, n, (r, nb), device=_DEV, generator=g).to(torch.int32))
        st["bias"] = _Held(3 * torch.randn(r, nb, device=_DEV, generator=g))
        st["bias_n"] = _Held(_words([max(0, nb - 3 * (i % 5)) for i in range(r)]))
    if case["mask"]:
        words = -(-n // 32)
        # a grammar allows a few tokens in some states and almost all of them inside a string
        wide = torch.rand(r, 1, device=_DEV, generator=g) < 0.5
        few = torch.randint(-2**31, 2**31, (r, words), device=_DEV, generator=g, dtype=torch.int64)
        few = few & torch.randint(-2**31, 2**31, (r, words), device=_DEV, generator=g, dtype=torch.int64)
        st["mask"] = _Held(torch.where(wide, torch.full_like(few, -1), few).to(torch.int32))
    if own:
        from tuckmill_b200 import cuda
        st["partial"] = _Storage.take(r * cuda.LOGITS_PARTIAL_BYTES)
    return st


# ---- one pass -------------------------------------------------------------------------------------


def run(state):
    return {"attention": _run_attention, "evict": _run_evict, "copy": _run_copy, "choose": _run_choose}[state["case"]["kind"]](state)


def _norm_rope(x, w, pos, inv_freq, eps=1e-6):
    """x [S][heads][hd] normed, weighted and rotated at each sequence's position."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = inv_freq.numel()
    angle = (pos.float()[:, None] * inv_freq)[:, None, :]  # an f32 product, as in the framework's other rotations
    c, s = angle.cos(), angle.sin()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def _run_attention(st):
    c = st["case"]
    s, heads, kvh, hd, page = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    scale = 1.0 / math.sqrt(hd)
    w_in, w_out = st.get("weights"), st.get("weights_out")
    result = {"out": st["out"].t, "k": st["k"].t, "v": st["v"].t}
    if w_out:
        result["weights"] = w_out.t
    if own:
        q, k, v = st["views"]
        width = (heads + 2 * kvh) * hd
        st["ctx"].attention_decode_paged(q, k, v, st["q_norm"].b, st["k_norm"].b, st["inv_freq"].b, st["k"].b, st["v"].b,
                                         st["table"].b, st["out"].b, st["scratch"].b, st["pos"].b, st["lens"].b,
                                         st["status"].b, s, heads, kvh, hd, c["n_rot"], st["pages"], page, st["max_pages"],
                                         c["window"], 1e-6, scale, q_stride=width, kv_stride=width,
                                         weights_in=w_in.b if w_in else None, weights_out=w_out.b if w_out else None)
        return result
    qkv, lens, table = st["qkv"].t.view(s, heads + 2 * kvh, hd), st["lens"].t.long(), st["table"].t.long()
    q = _norm_rope(qkv[:, :heads], st["q_norm"].t, st["pos"].t, st["inv_freq"].t)
    k = _norm_rope(qkv[:, heads:heads + kvh], st["k_norm"].t, st["pos"].t, st["inv_freq"].t)
    at = torch.gather(table, 1, (lens // page)[:, None])[:, 0]
    st["k"].t[at, :, lens % page] = k.half()
    st["v"].t[at, :, lens % page] = qkv[:, heads + kvh:].half()
    j = torch.arange(st["max_pages"] * page, device=_DEV)[None, :]
    seen = j <= lens[:, None]
    if c["window"]:
        seen = seen & (j + c["window"] > lens[:, None])
    ids = table.clamp(min=0)
    hide = ~seen[:, None, :, None]
    rows = lambda pool: pool[ids].permute(0, 2, 1, 3, 4).reshape(s, kvh, -1, hd).float().masked_fill(hide, 0)  # noqa: E731
    scores = torch.matmul(q.view(s, kvh, heads // kvh, hd), rows(st["k"].t).transpose(-1, -2)) * scale
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    st["out"].t.copy_(torch.matmul(p, rows(st["v"].t)).view(s, heads * hd))
    if w_out:
        before = torch.where((j < lens[:, None])[:, None, :], w_in.t, 0.0)  # the new row has drawn nothing yet
        w_out.t.copy_(torch.where((j <= lens[:, None])[:, None, :], before + p.sum(2), w_out.t))
    return result


def _run_evict(st):
    c = st["case"]
    page, keep, first, recent = c["page"], c["keep"], c["first"], c["recent"]
    result = {n: st[n].t for n in ("k", "v", "weights_out", "kept", "lens_out")}
    if own:
        st["ctx"].kv_pages_evict(st["k"].b, st["v"].b, st["table"].b, st["to"].b, st["lens"].b, st["lens_out"].b,
                                 st["weights"].b, st["weights_out"].b, st["kept"].b, st["status"].b, c["seqs"],
                                 c["kv_heads"], c["head_dim"], st["pages"], page, st["max_pages"], keep, first, recent)
        return result
    lens, w = st["lens"].t.long()[:, None, None], st["weights"].t
    j = torch.arange(w.shape[-1], device=_DEV).expand_as(w)
    held = (j < first) | (j >= lens - recent)  # rows that stay whatever they drew
    rank = torch.where(j >= lens, -1, torch.where(held | (lens <= keep), 1, 0))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    order = torch.gather(order, -1, torch.sort(torch.gather(rank, -1, order), dim=-1, descending=True, stable=True).indices)
    chosen = torch.sort(torch.where(torch.gather(j, -1, order[..., :keep]) < lens, order[..., :keep], 1 << 30), dim=-1).values
    i = torch.arange(keep, device=_DEV).expand_as(chosen)
    live = i < lens
    st["kept"].t.copy_(torch.where(live, chosen, _NONE))
    st["lens_out"].t.copy_(torch.clamp(st["lens"].t, max=keep))
    src, dst = torch.where(live, chosen, chosen[..., :1]), torch.where(live, i, 0)  # the rest writes the first row again
    h = torch.arange(c["kv_heads"], device=_DEV)[None, :, None]
    seq = torch.arange(c["seqs"], device=_DEV)[:, None, None]
    a, b = st["table"].t.long()[seq, src // page], st["to"].t.long()[seq, dst // page]
    for pool in (st["k"].t, st["v"].t):
        pool[b, h, dst % page] = pool[a, h, src % page]
    st["weights_out"].t[..., :keep] = torch.where(live, torch.gather(w, -1, src), st["weights_out"].t[..., :keep])
    return result


def _run_copy(st):
    c = st["case"]
    page, to_pages = c["page"], c["to_pages"]
    if own:
        st["ctx"].kv_pages_copy(st["kc"].b, st["vc"].b, st["k"].b, st["v"].b, st["table"].b, st["status"].b, st["pages"],
                                page, st["max_pages"], c["kv_heads"], c["head_dim"], st["cap"], to_pages, st["runs"])
    else:
        runs = st["runs_dev"]
        of = torch.repeat_interleave(torch.arange(len(st["runs"]), device=_DEV), runs[:, 3], output_size=st["rows"])
        first = torch.cumsum(runs[:, 3], 0) - runs[:, 3]
        row = torch.arange(st["rows"], device=_DEV) - first[of] + runs[of, 2]
        seq, at = runs[of, 0], st["table"].t.long()[runs[of, 1], row // page]
        for dense, pool in ((st["kc"].t, st["k"].t), (st["vc"].t, st["v"].t)):
            if to_pages:
                pool[at, :, row % page] = dense[seq, :, row]
            else:
                dense[seq, :, row] = pool[at, :, row % page]
    return {n: st[n].t for n in (("k", "v") if to_pages else ("kc", "vc"))}


def _run_choose(st):
    c = st["case"]
    r, n, stride = c["rows"], c["vocab"], st["stride"]
    result = {"y": st["y"].t, "log": st["log"].t}
    get = lambda name: st[name].b if name in st else None  # noqa: E731
    if own:
        st["ctx"].logits_adjust_rows(st["x"].b, st["y"].b, r, n, st["log"].b, stride, 1, st["pos"].b, st["pen"].b,
                                     prompt_len=st["prompt"].b, bias_ids=get("bias_ids"), bias_values=get("bias"),
                                     bias_count=get("bias_n"), bias_cap=c["biases"], mask=get("mask"), partial=st["partial"].b)
        return result
    x, log = st["x"].t, st["log"].t.long().clamp(min=0)
    end, start = st["pos"].t.long()[:, None] + 1, st["prompt"].t.long()[:, None]
    j = torch.arange(stride, device=_DEV)[None, :]
    count = torch.zeros(r, n, device=_DEV).scatter_add_(1, log, ((j >= start) & (j < end)).float())
    seen = torch.zeros(r, n, device=_DEV).scatter_add_(1, log, (j < end).float()) > 0
    rep, presence, freq = (st["pen"].t[:, i:i + 1] for i in range(3))
    y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    y = torch.where(count > 0, y - freq * count - presence, y)
    if "bias" in st:  # a token that is named twice gets the later value
        nb = c["biases"]
        e = torch.arange(1, nb + 1, device=_DEV).expand(r, nb)
        e = torch.where(e <= st["bias_n"].t.long()[:, None], e, 0)
        last = torch.zeros(r, n, dtype=torch.int64, device=_DEV).scatter_reduce_(1, st["bias_ids"].t.long(), e, "amax")
        y = torch.where(last > 0, y + torch.gather(st["bias"].t, 1, (last - 1).clamp(min=0)), y)
    if "mask" in st:
        bit = torch.arange(32, device=_DEV)
        allowed = ((st["mask"].t[:, :, None] >> bit) & 1).bool().view(r, -1)[:, :n]
    else:
        allowed = torch.ones_like(x, dtype=torch.bool)
    y = torch.where(allowed, y, -math.inf)
    st["y"].t.copy_(y)
    can = allowed & ~y.isnan()
    best = torch.where(can, y, -math.inf).amax(-1, keepdim=True)
    ids = torch.where(can & (y == best), torch.arange(n, device=_DEV), 1 << 40).amin(-1, keepdim=True)
    st["log"].t.scatter_(1, end, torch.where(ids < n, ids, _NONE).to(torch.int32))
    return result


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "evict": _exact_evict, "copy": _exact_copy, "choose": _exact_choose}[case["kind"]](case, st)


def _rotated(x, w, pos, inv_freq):
    """One head vector of f64: x / rms(x) * w, pairs (i, i + half) turned by the f32 angle pos * inv_freq[i]."""
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
    angle = (torch.tensor(float(pos), dtype=torch.float32, device=_DEV) * inv_freq).double()
    half = inv_freq.numel()
    y = x.clone()
    y[..., :half] = x[..., :half] * torch.cos(angle) - x[..., half:2 * half] * torch.sin(angle)
    y[..., half:2 * half] = x[..., :half] * torch.sin(angle) + x[..., half:2 * half] * torch.cos(angle)
    return y


def _exact_attention(case, st):
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = heads // kvh
    pk, pv = st["k"].t.clone(), st["v"].t.clone()
    out = torch.zeros(case["seqs"], heads, hd, dtype=torch.float64, device=_DEV)
    weights = st["weights_out"].t.double() if case["weights"] else None
    for s, n in enumerate(_lengths(case)):
        x = st["qkv"].t[s].view(-1, hd).double()
        pos = n + case["dropped"]
        q = _rotated(x[:heads], st["q_norm"].t, pos, st["inv_freq"].t)
        ids = st["table"].t[s, : n // page + 1].long()
        last = int(ids[-1])
        pk[last, :, n % page] = _rotated(x[heads:heads + kvh], st["k_norm"].t, pos, st["inv_freq"].t).half()
        pv[last, :, n % page] = x[heads + kvh:].half()
        lo = max(0, n + 1 - case["window"]) if case["window"] else 0
        p0 = lo // page
        for h in range(kvh):
            keys = pk[ids[p0:], h].reshape(-1, hd)[lo - p0 * page: n + 1 - p0 * page].double()
            vals = pv[ids[p0:], h].reshape(-1, hd)[lo - p0 * page: n + 1 - p0 * page].double()
            e = torch.softmax(q[h * group:(h + 1) * group] @ keys.T / math.sqrt(hd), -1)
            out[s, h * group:(h + 1) * group] = e @ vals
            if weights is not None:
                weights[s, h, :n] = st["weights"].t[s, h, :n].double()
                weights[s, h, n] = 0
                weights[s, h, lo:n + 1] += e.sum(0)
    got = {"out": out.view(case["seqs"], -1), "k": pk.double(), "v": pv.double()}
    if weights is not None:
        got["weights"] = weights
    return got


def _exact_evict(case, st):
    page, keep = case["page"], case["keep"]
    pk, pv, w = st["k"].t.double(), st["v"].t.double(), st["weights"].t.cpu().numpy().astype(np.float64)
    w_out = np.zeros_like(w)
    kept = np.full((case["seqs"], case["kv_heads"], keep), _NONE, np.int64)
    lens = _lengths(case)
    table, to = st["table"].t.cpu().numpy(), st["to"].t.cpu().numpy()
    for s, n in enumerate(lens):
        for h in range(case["kv_heads"]):
            if n <= keep:
                chosen = np.arange(n)
            else:
                middle = np.arange(case["first"], n - case["recent"])
                most = middle[np.lexsort((middle, -w[s, h, middle]))][: keep - case["first"] - case["recent"]]
                chosen = np.sort(np.concatenate([np.arange(case["first"]), most, np.arange(n - case["recent"], n)]))
            m = len(chosen)
            kept[s, h, :m], w_out[s, h, :m] = chosen, w[s, h, chosen]
            a, b = torch.from_numpy(table[s, chosen // page]).to(_DEV).long(), torch.from_numpy(to[s, np.arange(m) // page]).to(_DEV).long()
            ra, rb = torch.from_numpy(chosen % page).to(_DEV), torch.from_numpy(np.arange(m) % page).to(_DEV)
            for pool in (pk, pv):
                pool[b, h, rb] = pool[a, h, ra]
    return {"k": pk, "v": pv, "weights_out": w_out, "kept": kept, "lens_out": np.minimum(lens, keep)}


def _exact_copy(case, st):
    page = case["page"]
    k, v, kc, vc = (st[n].t.double() for n in ("k", "v", "kc", "vc"))
    table = st["table"].t.cpu().numpy()
    for seq, at, lo, n in st["runs"]:
        for p in range(lo // page, (lo + n - 1) // page + 1):
            a, b = max(lo, p * page), min(lo + n, (p + 1) * page)
            for dense, pool in ((kc, k), (vc, v)):
                rows = pool[int(table[at, p]), :, a - p * page:b - p * page]
                if case["to_pages"]:
                    rows.copy_(dense[seq, :, a:b])
                else:
                    dense[seq, :, a:b] = rows
    return {"k": k, "v": v} if case["to_pages"] else {"kc": kc, "vc": vc}


def _exact_choose(case, st):
    y = st["x"].t.double().cpu().numpy()
    log, pos, prompt, pen = (st[n].t.cpu().numpy() for n in ("log", "pos", "prompt", "pen"))
    for r in range(case["rows"]):
        end = pos[r] + 1
        rep, presence, freq = (float(v) for v in pen[r])
        seen = np.unique(log[r, :end])
        y[r, seen] = np.where(y[r, seen] > 0, y[r, seen] / rep, y[r, seen] * rep)
        ids, times = np.unique(log[r, prompt[r]:end], return_counts=True)
        y[r, ids] -= presence + freq * times
        if case["biases"]:
            m = int(st["bias_n"].t[r])
            named = dict(zip(st["bias_ids"].t[r, :m].tolist(), st["bias"].t[r, :m].tolist()))
            if named:
                y[r, list(named)] += list(named.values())
        if case["mask"]:
            words = st["mask"].t[r].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[: case["vocab"]]
            y[r, bits == 0] = -np.inf
    return {"y": y, "log": None}  # the choice is a whole number: it has no value in 64 bits of its own
