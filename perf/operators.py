"""The operators of a serving and scoring step on the engine, as cases that can
be timed and compared: keys and values appended to a paged cache with their
rotation, the attention of one new token per sequence over that cache, and the
log probabilities of given tokens with entropy and top alternatives, forward
and backward.

`listed()` names the cases, `draw(rng)` gives more of the same ranges,
`prepare(case, seed)` makes what a program holds before the call, `run(state)`
is one pass, `work(case)` its unavoidable bytes and operations and
`exact(case, seed)` the outputs in 64 bits.

Where `own` is false, `run` computes an operator in elementary torch
operations in 32 bits.  Where it is true, it makes the engine's calls
(metalium-rs_amd/miburn.py over include/miburn.h) on buffers that hold the same
values: the engine works on buffers of its own, so `prepare` uploads the inputs
as they are, with no cast and no other layout.  Results stay on the device, as
in a program that feeds them to the next call: `run` then returns tensors that
name their engine buffers and read them back when they are looked at.

A page holds `page` consecutive positions of one sequence: row
(p * kv + j) * page + o of the pools is offset o of page p for key/value head
j.  A sequence's row of the page table names its pages in order, -1 behind
them; its length counts the new positions.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROPE_THETA = 100000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# (heads, kv heads, head width): the decoders of this repository's benchmark
# and cases, and generic ones beside them: one head per kv head, twelve, one
# kv head for all, narrow and wide heads.
HEADS = ((9, 3, 64), (16, 4, 64), (8, 8, 64), (32, 8, 128), (24, 2, 128), (12, 1, 128), (4, 2, 32), (40, 8, 128))
PAGES = (16, 16, 64, 32, 8, 48)
MOST = 400 << 20  # bytes a drawn case may move


def listed():
    return [
        # One decode step's new rows of 32 sequences: rotated and stored, a
        # call that latency bounds.
        dict(name="append_b32", kind="append", seqs=32, new=1, ctx=300, ragged=True, heads=32, kv=8, d=128, page=16,
             rows="f32", cache="bf16", out="f32"),
        # Five prompts of unequal lengths, one behind the other, on top of what
        # their sequences hold already (a chunk of a long prompt each).
        dict(name="append_prompts", kind="append", seqs=5, new=1201, ctx=700, ragged=True, heads=9, kv=3, d=64,
             page=64, rows="f32", cache="f32", out="f32"),
        # One sequence's decode step after a 512-token prompt: latency.
        dict(name="attend_b1", kind="attend", seqs=1, ctx=577, ragged=False, heads=9, kv=3, d=64, page=16, q="f32",
             cache="f32", out="f32"),
        # A full decode batch of unequal lengths, idle slots among them.
        dict(name="attend_b32", kind="attend", seqs=32, ctx=1000, ragged=True, heads=9, kv=3, d=64, page=16, q="f32",
             cache="f32", out="f32"),
        # Seven sequences with twelve query heads a kv head, in pages that
        # are no power of two; BF16 in and out.
        dict(name="attend_b7", kind="attend", seqs=7, ctx=9001, ragged=True, heads=24, kv=2, d=128, page=48, q="bf16",
             cache="bf16", out="bf16"),
        # One very long context: the work has to be split over it.
        dict(name="attend_long", kind="attend", seqs=1, ctx=100001, ragged=False, heads=32, kv=8, d=128, page=64,
             q="f32", cache="bf16", out="f32"),
        # A large serving batch of unequal lengths.
        dict(name="attend_b64", kind="attend", seqs=64, ctx=4000, ragged=True, heads=32, kv=8, d=128, page=16,
             q="f32", cache="bf16", out="f32"),
        # The answer to one request's token, with five alternatives: latency.
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=49152, logits="f32", top=5, scale=1.0),
        # A serving batch's, at a temperature of 0.7, with twenty.
        dict(name="logprobs_64", kind="logprobs", rows=64, vocab=49152, logits="bf16", top=20, scale=1 / 0.7),
        # Scoring a text: every position's token.
        dict(name="logprobs_2001", kind="logprobs", rows=2001, vocab=49152, logits="f32", top=5, scale=1.0),
        # Training on log probabilities and entropy: the transformer's
        # vocabulary, and an odd one in BF16.
        dict(name="backward_8192", kind="backward", rows=2048, vocab=8192, logits="f32", out="f32", scale=1.0),
        dict(name="backward_odd", kind="backward", rows=1001, vocab=40001, logits="bf16", out="bf16", scale=1 / 0.7),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm: odd ones as
    often as even, one in three rounded down to a multiple of 64 or 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((1, 1, 1, 1, 8, 64)) if hi > 64 else 1
    return min(hi, max(lo, v // step * step if v >= step else v))


def draw(rng):
    kind = rng.choice(("append", "append", "attend", "attend", "attend", "logprobs", "logprobs", "backward"))
    if kind in ("append", "attend"):
        heads, kv, d = rng.choice(HEADS)
        cache = rng.choice(("f32", "bf16", "bf16"))
        c = dict(kind=kind, heads=heads, kv=kv, d=d, page=rng.choice(PAGES), cache=cache, ragged=rng.random() < 0.7)
        types = ("f32", "f32", "bf16")
        if kind == "append":
            new = 1 if rng.random() < 0.5 else _between(rng, 2, 1500)
            most = max(1, min(256 if new == 1 else 16, 8000 // new))
            return dict(c, seqs=_between(rng, 1, most), new=new, ctx=_between(rng, 1, 1000), rows=rng.choice(types),
                        out=rng.choice(types))
        seqs = _between(rng, 1, 200)
        most = MOST // (2 * seqs * kv * d * (4 if cache == "f32" else 2))
        return dict(c, seqs=seqs, ctx=_between(rng, 1, min(120000, max(2, most))), q=rng.choice(types),
                    out=rng.choice(types))
    vocab = _between(rng, 500, 160000)
    rows = _between(rng, 1, max(2, min(8000, MOST // ((4 if kind == "logprobs" else 8) * vocab))))
    c = dict(kind=kind, rows=rows, vocab=vocab, logits=rng.choice(("f32", "bf16")),
             scale=rng.choice((1.0, 1.0, 1 / 0.7, 0.5)))
    return dict(c, top=rng.choice((0, 1, 5, 20, 32))) if kind == "logprobs" else dict(c, out=rng.choice(("f32", "bf16")))


# ------------------------------------------------------------------ inputs


def _spread(case, n, hi):
    """n lengths of [1, hi] spread evenly in a shuffled order where the case
    is ragged, else n times hi."""
    if not case["ragged"]:
        return [hi] * n
    return [1 + int((hi - 1) * ((0.37 + 0.6180339887498949 * i) % 1.0)) for i in range(n)]


def _news(case):
    """The new rows of each sequence of an append."""
    return [1] * case["seqs"] if case["new"] == 1 else _spread(case, case["seqs"], case["new"])


def _lens(case):
    """The sequences' lengths, the new positions counted; in a ragged batch of
    attention rows every sixteenth slot is idle (length 0)."""
    if case["kind"] == "append":
        return [a + b - 1 for a, b in zip(_spread(case, case["seqs"], case["ctx"]), _news(case))]
    lens = _spread(case, case["seqs"], case["ctx"])
    return [0 if case["ragged"] and i % 16 == 9 else n for i, n in enumerate(lens)]


def _page_table(case, lens, g):
    """The pool's pages and the table naming them: a shuffled pool, a few
    pages more than the sequences hold, -1 behind a sequence's last page."""
    need = [-(-n // case["page"]) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return total, table


def _rope_tables(n, d):
    freq = ROPE_THETA ** (-2.0 * np.arange(d // 2) / d)
    ang = np.arange(n)[:, None] * freq[None, :]
    cos, sin = np.cos(ang), np.sin(ang)
    return (torch.from_numpy(np.concatenate([cos, cos], 1)).float().cuda(),
            torch.from_numpy(np.concatenate([-sin, sin], 1)).float().cuda())


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, of="f32"):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(TYPES[of])

    def column(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda").reshape(-1, 1)
    kind = case["kind"]
    if kind in ("append", "attend"):
        heads, kv, d, lens = case["heads"], case["kv"], case["d"], _lens(case)
        pages, table = _page_table(case, lens, g)
        t = dict(k=normal(pages * kv * case["page"], d, of=case["cache"]),
                 v=normal(pages * kv * case["page"], d, of=case["cache"]), table=table, lens=column(lens))
        if kind == "attend":
            return dict(t, q=normal(len(lens), heads * d, of=case["q"]))
        cos, sin = _rope_tables(max(lens), d)
        starts = np.concatenate([[0], np.cumsum(_news(case))]).tolist()
        t.update(qkv=normal(starts[-1], (heads + 2 * kv) * d, of=case["rows"]), cos=cos, sin=sin)
        return t if case["new"] == 1 else dict(t, starts=column(starts))
    rows, vocab = case["rows"], case["vocab"]
    # A trained head's logits: a few well above a broad rest.
    x = normal(rows, vocab, std=2.0)
    x += 3.0 * (normal(rows, vocab) > 3.0)
    t = dict(logits=x.to(TYPES[case["logits"]]),
             targets=torch.randint(0, vocab, (rows, 1), generator=g, device="cuda", dtype=torch.int32))
    if kind == "backward":  # what the forward pass left, and the loss's gradients
        z = t["logits"].double() * case["scale"]
        lse = torch.logsumexp(z, 1, keepdim=True)
        entropy = lse - (torch.exp(z - lse) * z).sum(1, keepdim=True)
        t.update(lse=lse.float(), entropy=entropy.float(), d_logp=normal(rows, 1, std=1.0 / rows),
                 d_entropy=normal(rows, 1, std=0.01 / rows))
    return t


# ------------------------------------------------------------------- state

_ENGINE = None


def _engine():
    """The process's engine: a program attaches to the device once."""
    global _ENGINE
    if _ENGINE is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "metalium-rs_amd"))
        import miburn
        _ENGINE = miburn.Engine(0)
    return _ENGINE


class Result(torch.Tensor):
    """A result on the device: reading it in any way reads its buffer back."""

    @staticmethod
    def of(read):
        t = torch.empty(0).as_subclass(Result)
        t.read = read
        return t

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        def real(v):
            return v.read() if isinstance(v, Result) else v
        return func(*[real(a) for a in args], **{k: real(v) for k, v in (kwargs or {}).items()})


class Buffers:
    """What a program on the engine holds: input buffers, and the last pass's
    results (freed when the next pass replaces them)."""

    def __init__(self, tensors):
        self.eng, self.ids, self.out, self.results = _engine(), {}, {}, {}
        for name, t in tensors.items():
            host = t.cpu()
            if t.dtype == torch.bfloat16:
                self.ids[name] = self.eng.upload_bf16(host.view(torch.int16).numpy().view(np.uint16))
            elif t.dtype == torch.int32:
                self.ids[name] = self.eng.upload_i32(host.numpy())
            else:
                self.ids[name] = self.eng.upload(host.numpy())

    def _read(self, name):
        host = self.eng.download(self.out[name] if name in self.out else self.ids[name])
        if host.dtype == np.uint16:
            return torch.from_numpy(host.view(np.int16)).view(torch.bfloat16)
        return torch.from_numpy(host)

    def give(self, *held, **out):
        """The pass's results, in the place of the last one's; `held` names
        buffers of the program's own that the pass updated."""
        for id_ in self.out.values():
            self.eng.free(id_)
        self.out = out
        if not self.results:
            for name in (*held, *out):
                self.results[name] = Result.of(lambda name=name: self._read(name))
        return self.results

    def __del__(self):
        if self.eng.ctx:
            for id_ in list(self.out.values()) + list(self.ids.values()):
                self.eng.free(id_)


def prepare(case, seed):
    tensors = _inputs(case, seed)
    return case, Buffers(tensors) if own else tensors


# --------------------------------------------------------------------- run


def run(state):
    case, held = state
    if own:
        return _run_own(case, held)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs, "backward": _backward}[case["kind"]](case, held)


def _run_own(c, b):
    e, i = b.eng, b.ids
    elem = {"f32": 0, "bf16": 3}  # the binding's F32 and BF16
    if c["kind"] == "append":
        q = e.qkv_rope_paged(i["qkv"], i["cos"], i["sin"], i["table"], i["lens"], i.get("starts", 0), c["heads"],
                             c["kv"], c["page"], i["k"], i["v"], elem[c["out"]])
        return b.give("k", "v", q=q)
    if c["kind"] == "attend":
        return b.give(out=e.paged_attention(i["q"], i["k"], i["v"], i["table"], i["lens"], c["heads"], c["kv"],
                                            c["page"], c["d"] ** -0.5, elem[c["out"]]))
    if c["kind"] == "logprobs":
        r = e.token_logprobs(i["logits"], i["targets"], c["scale"], c["top"])
        out = dict(logp=r.logp, lse=r.lse, entropy=r.entropy)
        return b.give(**out, top_logp=r.top_logp, top_ids=r.top_ids) if c["top"] else b.give(**out)
    return b.give(dlogits=e.token_logprobs_backward(i["logits"], i["targets"], i["lse"], i["entropy"], i["d_logp"],
                                                    i["d_entropy"], c["scale"], elem[c["out"]]))


def _append(c, t):
    heads, kv, d, page = c["heads"], c["kv"], c["d"], c["page"]
    rows, lens = t["qkv"].shape[0], t["lens"].reshape(-1).long()
    at = torch.arange(rows, device="cuda")
    if "starts" in t:
        ends = t["starts"].reshape(-1)[1:].long()
        seq = torch.searchsorted(ends, at, right=True)
        pos = lens[seq] - ends[seq] + at
    else:
        seq, pos = at, lens - 1
    x = t["qkv"].float().reshape(rows, heads + 2 * kv, d)
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    turned = torch.cat([qk[..., d // 2:], qk[..., :d // 2]], -1)
    qk = qk * t["cos"][pos][:, None] + turned * t["sin"][pos][:, None]
    slot = (t["table"][seq, pos // page].long()[:, None] * kv + torch.arange(kv, device="cuda")) * page + (pos % page)[:, None]
    t["k"][slot] = qk[:, heads:].to(t["k"].dtype)
    t["v"][slot] = v.to(t["v"].dtype)
    return dict(k=t["k"], v=t["v"], q=qk[:, :heads].reshape(rows, heads * d).to(TYPES[c["out"]]))


def _attend(c, t):
    heads, kv, d, page = c["heads"], c["kv"], c["d"], c["page"]
    seqs, per = t["table"].shape
    pages = t["table"].clamp(min=0).long()

    def rows_of(pool):
        return pool.reshape(-1, kv, page, d)[pages].permute(0, 2, 1, 3, 4).reshape(seqs * kv, per * page, d).float()
    q = t["q"].float().reshape(seqs * kv, heads // kv, d).transpose(1, 2).contiguous()
    s = torch.matmul(rows_of(t["k"]), q) * d ** -0.5
    hidden = torch.arange(per * page, device="cuda")[None, :, None] >= t["lens"].long().repeat_interleave(kv, 0)[:, :, None]
    s = s.masked_fill(hidden, -math.inf)
    e = torch.exp(s - s.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    p = (e / e.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)).transpose(1, 2).contiguous()
    return dict(out=torch.matmul(p, rows_of(t["v"])).reshape(seqs, heads * d).to(TYPES[c["out"]]))


def _logprobs(c, t):
    x = t["logits"].float()
    z = x * c["scale"]
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = z.amax(1, keepdim=True) + torch.log(total)
    entropy = torch.log(total) - (e * d).sum(1, keepdim=True) / total
    out = dict(logp=z.gather(1, t["targets"].long()) - lse, lse=lse, entropy=entropy)
    if c["top"]:
        # Value and column in one whole number, no two alike: the larger value
        # first, the lower column among equals (-0 and 0 are equal).
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
        key = (key << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device="cuda"))
        ids = torch.topk(key, c["top"], 1).values
        ids = 0x7FFFFFFF - (ids & 0xFFFFFFFF)
        out.update(top_logp=z.gather(1, ids) - lse, top_ids=ids.int())
    return out


def _backward(c, t):
    logp = t["logits"].float() * c["scale"] - t["lse"]
    p = torch.exp(logp)
    g = -p * (t["d_logp"] + t["d_entropy"] * (logp + t["entropy"]))
    g.scatter_add_(1, t["targets"].long(), t["d_logp"])
    return dict(dlogits=(g * c["scale"]).to(TYPES[c["out"]]))


# -------------------------------------------------------------------- work


def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    c = case
    if c["kind"] == "append":
        rows, h = sum(_news(c)), c["heads"] + 2 * c["kv"]
        moved = rows * c["d"] * (h * _bytes(c["rows"]) + c["heads"] * _bytes(c["out"]) + 2 * c["kv"] * _bytes(c["cache"]))
        return dict(bytes=moved + 8 * c["d"] * min(rows, max(_lens(c))) + 4 * (rows + c["seqs"]),
                    flops=3 * rows * c["d"] * (c["heads"] + c["kv"]))
    if c["kind"] == "attend":
        total = sum(_lens(c))
        moved = 2 * total * c["kv"] * c["d"] * _bytes(c["cache"])
        moved += c["seqs"] * c["heads"] * c["d"] * (_bytes(c["q"]) + _bytes(c["out"]))
        return dict(bytes=moved + 4 * (total // c["page"] + 2 * c["seqs"]), flops=4 * total * c["heads"] * c["d"])
    n = c["rows"] * c["vocab"]
    if c["kind"] == "logprobs":
        return dict(bytes=n * _bytes(c["logits"]) + c["rows"] * (16 + 8 * c["top"]), flops=6 * n)
    return dict(bytes=n * (_bytes(c["logits"]) + _bytes(c["out"])) + 20 * c["rows"], flops=7 * n)


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    f = {n: x.double() if x.is_floating_point() else x.long() for n, x in t.items()}
    if c["kind"] == "append":
        return _exact_append(c, t, f)
    if c["kind"] == "attend":
        return _exact_attend(c, f)
    logp = torch.log_softmax(f["logits"] * c["scale"], 1) if c["kind"] == "logprobs" else None
    if logp is not None:
        lse = f["logits"][:, :1] * c["scale"] - logp[:, :1]
        out = dict(logp=logp.gather(1, f["targets"]), lse=lse, entropy=-(logp.exp() * logp).sum(1, keepdim=True))
        if c["top"]:
            best = torch.sort(f["logits"], dim=1, descending=True, stable=True)
            out.update(top_logp=best.values[:, :c["top"]] * c["scale"] - lse, top_ids=best.indices[:, :c["top"]].int())
        return out
    # d(logp_t)/dz_j = [j = t] - p_j and dH/dz_j = -p_j (logp_j + H), z the scaled logits.
    logp = f["logits"] * c["scale"] - f["lse"]
    p, one = logp.exp(), torch.zeros_like(logp).scatter_(1, f["targets"], 1.0)
    grad = f["d_logp"] * (one - p) - f["d_entropy"] * p * (logp + f["entropy"])
    return dict(dlogits=c["scale"] * grad)


def _exact_append(c, t, f):
    heads, kv, d, page = c["heads"], c["kv"], c["d"], c["page"]
    k, v, q, row = f["k"].clone(), f["v"].clone(), [], 0
    for s, (n, new) in enumerate(zip(_lens(c), _news(c))):
        pos = torch.arange(n - new, n, device="cuda")
        x = f["qkv"][row:row + new].reshape(new, -1, d)
        row += new
        # Each pair (i, i + d / 2) turned by its angle.
        a, b = x[..., :d // 2], x[..., d // 2:]
        co, si = f["cos"][pos][:, None, :d // 2], f["sin"][pos][:, None, d // 2:]
        turned = torch.cat([a * co - b * si, b * co + a * si], -1)
        q.append(turned[:, :heads].reshape(new, heads * d))
        for j in range(kv):
            at = (f["table"][s][pos // page] * kv + j) * page + pos % page
            k[at], v[at] = turned[:, heads + j], x[:, heads + kv + j]
    return dict(k=k, v=v, q=torch.cat(q))


def _exact_attend(c, f):
    heads, kv, d, page = c["heads"], c["kv"], c["d"], c["page"]
    out = torch.zeros(c["seqs"], heads, d, dtype=torch.float64, device="cuda")
    for s, n in enumerate(_lens(c)):
        if n == 0:
            continue
        pos = torch.arange(n, device="cuda")
        for j in range(kv):
            at = (f["table"][s][pos // page] * kv + j) * page + pos % page
            mine = slice(j * heads // kv, (j + 1) * heads // kv)
            p = torch.softmax(f["q"][s].reshape(heads, d)[mine] @ f["k"][at].T * d ** -0.5, 1)
            out[s, mine] = p @ f["v"][at]
    return dict(out=out.reshape(c["seqs"], heads * d))
