"""Operators around a paged key/value cache: plain forms, calls and workloads.

Four operators, each in its plain form (elementary torch operations) and, where
`own` is true, as calls of beacon_cuda:

- rope: rotary positions of token-major rows, interleaved or half pairs, on part
  of the head, with the scalings used for contexts longer than trained;
- qk_norm_rope: RMS norm of every query and key head, then the rotation;
- paged_append: new keys (rotated on the way) and values into cache pages;
- paged_attention: causal attention of queries over a paged cache, where groups
  of sequences share a prefix whose keys are read once for the group.

A case is a dict of plain values; `prepare` makes its tensors from the seed,
`run` is one pass, `exact` the same from the definition in 64 bits.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
# the scalings a case names: (scaling, theta, factor, original context)
SCALINGS = {
    "none": ("none", 500000.0, 1.0, 8192),
    "linear": ("linear", 10000.0, 4.0, 4096),
    "yarn": ("yarn", 10000.0, 8.0, 4096),
    "bands": ("bands", 500000.0, 8.0, 8192),
}
LOW_FREQ, HIGH_FREQ = 1.0, 4.0      # "bands": wavelengths per original context
BETA_FAST, BETA_SLOW = 32.0, 1.0    # "yarn": rotations per original context


def listed():
    return [
        # one new token of a small chat: only the launch and the latency count
        dict(name="rope-decode-1", op="rope", dtype="f32", tokens=1, heads=32, dim=128, rotary=128,
             layout="interleaved", scaling="none", context=4096),
        # queries of a long prompt chunk, half layout on three quarters of the head
        dict(name="rope-chunk-8192", op="rope", dtype="bf16", tokens=8192, heads=32, dim=128, rotary=96,
             layout="half", scaling="yarn", context=32768),
        # a decode batch: query and key norms with the rotation
        dict(name="norm-decode-8", op="qk_norm_rope", dtype="f32", tokens=8, heads=32, kv_heads=8, dim=128,
             rotary=128, layout="half", scaling="none", context=8192),
        # a prompt of odd length with many heads
        dict(name="norm-chunk-4099", op="qk_norm_rope", dtype="bf16", tokens=4099, heads=64, kv_heads=8, dim=128,
             rotary=128, layout="half", scaling="bands", context=65536),
        # decode step of 32 sequences: one row each, f32 projections into an f16 cache
        dict(name="append-decode-32", op="paged_append", dtype="f32", cache="f16", seqs=32, tokens=1, context=4096,
             kv_heads=8, dim=128, rotary=128, layout="interleaved", scaling="none", page=16),
        # ragged prompts appended behind what their sequences hold
        dict(name="append-prompts-7x1500", op="paged_append", dtype="bf16", cache="bf16", seqs=7, tokens=1500,
             context=2048, kv_heads=8, dim=128, rotary=128, layout="half", scaling="bands", page=32),
        # the smallest decode: one sequence, a short context, a small model's heads
        dict(name="attn-decode-1x257", op="paged_attention", dtype="f32", cache="f16", groups=1, seqs=1, prefix=0,
             suffix=257, new=1, heads=32, kv_heads=4, dim=64, page=16),
        # 32 requests behind one system prompt, f32 queries over the default f16 cache
        dict(name="attn-shared-32x4096", op="paged_attention", dtype="f32", cache="f16", groups=1, seqs=32,
             prefix=4096, suffix=512, new=1, heads=32, kv_heads=8, dim=128, page=16),
        # 64 samples of one long document
        dict(name="attn-shared-64x16384", op="paged_attention", dtype="bf16", cache="bf16", groups=1, seqs=64,
             prefix=16384, suffix=1024, new=1, heads=64, kv_heads=8, dim=128, page=32),
        # unrelated long conversations of different lengths: no prefix at all
        dict(name="attn-ragged-16x8192", op="paged_attention", dtype="f16", cache="f16", groups=16, seqs=1, prefix=0,
             suffix=8192, new=1, heads=32, kv_heads=8, dim=128, page=64),
        # eight beam searches of six beams, prompts that end inside a page
        dict(name="attn-beams-8x6x2049", op="paged_attention", dtype="f16", cache="f16", groups=8, seqs=6,
             prefix=2049, suffix=129, new=1, heads=32, kv_heads=8, dim=128, page=16),
        # four prompts, ragged, behind one shared prefix: prefill
        dict(name="attn-prompts-4x512", op="paged_attention", dtype="bf16", cache="bf16", groups=1, seqs=4,
             prefix=4096, suffix=512, new=512, heads=32, kv_heads=8, dim=128, page=16),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    caps = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    while True:
        op = rng.choice(["rope", "qk_norm_rope", "paged_append", "paged_attention", "paged_attention"])
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]))
        if op in ("rope", "qk_norm_rope"):
            c.update(tokens=_spread(rng, 1, 8192), heads=kv_heads * rng.choice([1, 2, 4, 7, 8]))
            if op == "qk_norm_rope":
                c.update(kv_heads=kv_heads)
        elif op == "paged_append":
            c.update(cache=c["dtype"] if c["dtype"] != "f32" else rng.choice(["f16", "bf16"]),
                     seqs=_spread(rng, 1, 64), tokens=_spread(rng, 1, 1500), kv_heads=kv_heads,
                     page=rng.choice([1, 8, 16, 24, 32, 64, 128]))
        if op != "paged_attention":
            c.update(dim=dim, rotary=rng.choice([dim, dim // 2, dim // 4 * 3]),
                     layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(sorted(SCALINGS)),
                     context=_spread(rng, 256, 65536 if op != "paged_append" else 4096))
        else:
            shared = rng.random() < 0.7
            new = 1 if rng.random() < 0.7 else _spread(rng, 2, 1024)
            c.update(cache="f16" if c["dtype"] == "f32" else c["dtype"], groups=_spread(rng, 1, 8 if shared else 32),
                     seqs=_spread(rng, 1, 64) if shared else 1, prefix=_spread(rng, 16, 16384) if shared else 0,
                     suffix=max(new, _spread(rng, 1, 1024 if shared else 16384)), new=new,
                     heads=kv_heads * rng.choice([1, 2, 4, 7, 8]), kv_heads=kv_heads, dim=dim,
                     page=rng.choice([8, 16, 24, 32, 64, 128]))
            if c["groups"] * c["seqs"] * (c["prefix"] + c["suffix"]) * kv_heads * dim > 1.2e9:
                continue  # the plain form reads every sequence's keys
        w = work(c)
        if all(w[m] <= caps[m] for m in caps):
            return c


# --- lengths and inputs ---------------------------------------------------------

def _ragged(n, lo, hi):
    """n lengths in [lo, hi], unlike each other, the last one hi."""
    f = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]
    f[-1] = 1.0
    return [lo + int(x * (hi - lo)) for x in f]


def _shape(c):
    """Per sequence: (new tokens, tokens behind the prefix, whole length)."""
    n = c["groups"] * c["seqs"]
    new = _ragged(n, max(1, c["new"] // 2), c["new"])
    tail = [max(a, b) for a, b in zip(new, _ragged(n, max(1, c["suffix"] // 4), c["suffix"]))]
    return new, tail, [c["prefix"] + t for t in tail]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed & 0x7FFFFFFF)

    def randn(*shape, dtype="f32", scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(DT[dtype])

    def ints(v):
        return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")

    s = {"case": c}
    if c["op"] in ("rope", "qk_norm_rope"):
        t = c["tokens"]
        # a decode batch stands anywhere; a prompt's tokens follow one another
        s["positions"] = ints(r.randint(0, c["context"], t) if t <= 256 else r.randint(0, c["context"]) + np.arange(t))
        s["q"] = randn(t, c["heads"], c["dim"], dtype=c["dtype"])
    if c["op"] == "qk_norm_rope":
        s["k"] = randn(c["tokens"], c["kv_heads"], c["dim"], dtype=c["dtype"], scale=2.0)
        s["qw"], s["kw"] = 1 + randn(c["dim"], scale=0.2), 1 + randn(c["dim"], scale=0.2)
    if c["op"] == "paged_append":
        b, page = c["seqs"], c["page"]
        held = r.randint(0, c["context"], b)
        new = np.array(_ragged(b, max(1, c["tokens"] // 2), c["tokens"]))
        rows = -(-(c["context"] + c["tokens"]) // page)
        pages = b * rows
        s["table"] = ints(r.permutation(pages).reshape(b, rows))
        s["seq_ids"] = ints(np.repeat(np.arange(b), new))
        s["positions"] = ints(np.concatenate([h + np.arange(n) for h, n in zip(held, new)]))
        t = int(new.sum())
        s["k"] = randn(t, c["kv_heads"], c["dim"], dtype=c["dtype"])
        s["v"] = randn(t, c["kv_heads"], c["dim"], dtype=c["dtype"])
        s["ck"] = randn(pages, page, c["kv_heads"], c["dim"], dtype=c["cache"])
        s["cv"] = randn(pages, page, c["kv_heads"], c["dim"], dtype=c["cache"])
    if c["op"] == "paged_attention":
        new, tail, lens = _shape(c)
        page, gs, prefix = c["page"], c["groups"], c["prefix"]
        shared = prefix // page                      # whole pages that a group shares
        rows = -(-max(lens) // page)
        own_rows = rows - shared
        pages = gs * shared + len(lens) * own_rows
        perm = r.permutation(pages)
        table = np.empty((len(lens), rows), dtype=np.int64)
        for i in range(len(lens)):
            k = i // c["seqs"]
            table[i, :shared] = perm[k * shared:(k + 1) * shared]
            table[i, shared:] = perm[gs * shared + i * own_rows:gs * shared + (i + 1) * own_rows]
        s["table"], s["lens"] = ints(table), ints(lens)
        s["starts"] = ints(np.concatenate([[0], np.cumsum(new)])) if c["new"] > 1 else None
        s["group_starts"] = ints(np.arange(gs + 1) * c["seqs"]) if prefix else None
        s["prefix_lens"] = ints([prefix] * gs) if prefix else None
        s["scale"] = c["dim"] ** -0.5
        s["max_new"], s["max_len"] = max(new), max(lens)  # the host's own bookkeeping
        s["q"] = randn(sum(new), c["heads"], c["dim"], dtype=c["dtype"], scale=1.5)
        s["ck"] = randn(pages, page, c["kv_heads"], c["dim"], dtype=c["cache"])
        s["cv"] = randn(pages, page, c["kv_heads"], c["dim"], dtype=c["cache"])
    return s


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e = size[c["dtype"]]
    if c["op"] in ("rope", "qk_norm_rope"):
        heads = c["heads"] + (c["kv_heads"] if c["op"] == "qk_norm_rope" else 0)
        n = c["tokens"] * heads * c["dim"]
        return {"bytes": 2 * n * e + 4 * c["tokens"], "flops": (7 if c["op"] == "qk_norm_rope" else 3) * n}
    if c["op"] == "paged_append":
        t = sum(_ragged(c["seqs"], max(1, c["tokens"] // 2), c["tokens"]))
        n = 2 * t * c["kv_heads"] * c["dim"]
        return {"bytes": n * (e + size[c["cache"]]) + 12 * t, "flops": 1.5 * n}
    new, tail, lens = _shape(c)
    keys = c["groups"] * c["prefix"] + sum(tail)
    # a row's keys: its sequence's up to its own position
    seen = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lens))
    bytes_ = 2 * sum(new) * c["heads"] * c["dim"] * e + 2 * keys * c["kv_heads"] * c["dim"] * size[c["cache"]]
    return {"bytes": bytes_ + 4 * -(-keys // c["page"]), "flops": 4 * seen * c["heads"] * c["dim"]}


# --- plain forms ------------------------------------------------------------------

def _turns(c, device):
    """The pairs' angles per position (64 bits) and the factor on sine and cosine."""
    kind, theta, factor, orig = SCALINGS[c["scaling"]]
    d = c["rotary"]
    i = torch.arange(0, d, 2, dtype=torch.float64, device=device)
    inv = theta ** (-i / d)
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "bands":
        waves = orig * inv / (2 * math.pi)           # turns in the original context
        mix = ((waves - LOW_FREQ) / (HIGH_FREQ - LOW_FREQ)).clamp(0, 1)
        return inv * (mix + (1 - mix) / factor), 1.0
    if kind == "yarn":
        def at(turns):
            return d * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(0, math.floor(at(BETA_FAST))), min(d - 1, math.ceil(at(BETA_SLOW)))
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv * (1 - ramp + ramp / factor), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _rotate(c, x, positions):
    """x [T, H, D] in 32 bits, its first `rotary` values rotated."""
    inv, scale = _turns(c, x.device)
    angle = positions.double()[:, None] * inv
    cos, sin = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    d = c["rotary"]
    rot, rest = x[..., :d], x[..., d:]
    if c["layout"] == "half":
        a, b = rot[..., :d // 2], rot[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = rot[..., 0::2], rot[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_attention(s):
    c = s["case"]
    b, most, page = c["groups"] * c["seqs"], s["max_len"], c["page"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    dev = s["q"].device
    seq = torch.arange(b, device=dev)
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(b + 1, device=dev)
    lens = s["lens"].long()
    # keys of the prefix are read through the group's first sequence
    pos = torch.arange(most, device=dev)
    through = torch.where(pos[None] < c["prefix"], (seq // c["seqs"] * c["seqs"])[:, None], seq[:, None])
    at = s["table"].long()[through, (pos // page)[None]]
    k = s["ck"][at, (pos % page)[None]].float().permute(0, 2, 3, 1)     # [b, hk, d, keys]
    v = s["cv"][at, (pos % page)[None]].float().permute(0, 2, 1, 3)     # [b, hk, keys, d]
    # every sequence's queries, padded to the longest
    j = torch.arange(s["max_new"], device=dev)
    new = starts[1:] - starts[:-1]
    live = j[None] < new[:, None]
    row = (starts[:-1, None] + j[None]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().reshape(b, -1, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(b, hk, -1, d), k).reshape(b, hk, h // hk, -1, most) * s["scale"]
    sees = pos[None, None] <= (lens - new)[:, None, None] + j[None, :, None]
    score = score.masked_fill(~sees[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, hk, -1, most), v).reshape(b, hk, h // hk, -1, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, -1, h, d)[live].to(s["q"].dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return _rotate(c, s["q"].float(), s["positions"]).to(s["q"].dtype)
    if c["op"] == "qk_norm_rope":
        return [_rotate(c, _norm(x.float(), w), s["positions"]).to(x.dtype)
                for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"]))]
    if c["op"] == "paged_append":
        p = s["positions"].long()
        at = s["table"].long()[s["seq_ids"].long(), p // c["page"]], p % c["page"]
        s["ck"][at] = _rotate(c, s["k"].float(), s["positions"]).to(s["ck"].dtype)
        s["cv"][at] = s["v"].to(s["cv"].dtype)
        return s["ck"], s["cv"]
    return _plain_attention(s)


# --- the framework's calls ----------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _backend():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "beacon-ai_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import beacon_cuda
    return beacon_cuda.CudaBackend(0), beacon_cuda._lib


_streams = {}


def _stream():
    """The framework's handle of torch's current stream, kept as a program keeps it."""
    raw = torch._C._cuda_getCurrentRawStream(0)  # (a Stream object costs microseconds)
    if raw not in _streams:
        _streams[raw] = _backend()[0].wrap_stream(raw)
    return _streams[raw]


@functools.lru_cache(maxsize=None)
def _rope_handle(scaling, rotary, layout):
    be, L = _backend()
    kind, theta, factor, orig = SCALINGS[scaling]
    kinds = {"none": L.ROPE_SCALING_NONE, "linear": L.ROPE_SCALING_LINEAR, "yarn": L.ROPE_SCALING_YARN,
             "bands": L.ROPE_SCALING_BANDS}
    return be.rope_create(theta=theta, rotary_dim=rotary, scaling=kinds[kind], factor=factor, original_context=orig,
                          layout=L.ROPE_HALF if layout == "half" else L.ROPE_INTERLEAVED)


def _handles(s):
    """The tensors of a state as the framework's, kept with it as a program keeps them."""
    if "handles" not in s:
        be, L = _backend()
        kind = {torch.float32: L.DTYPE_F32, torch.float16: L.DTYPE_F16, torch.bfloat16: L.DTYPE_BF16,
                torch.int32: L.DTYPE_I32}
        for name in ("q", "k"):
            if name in s and s["case"]["op"] != "paged_append":
                s["out_" + name] = torch.empty_like(s[name])
        s["handles"] = {n: be.wrap(x.data_ptr(), tuple(x.shape), kind[x.dtype]) for n, x in s.items()
                        if isinstance(x, torch.Tensor)}
        c = s["case"]
        s["rope"] = _rope_handle(c["scaling"], c["rotary"], c["layout"]) if "rotary" in c else None
    return s["handles"]


def _own(s):
    be, stream = _backend()[0], _stream()
    t = _handles(s)
    op = s["case"]["op"]
    if op == "rope":
        be.rope_scaled(stream, t["q"], t["positions"], s["rope"], out=t["out_q"])
        return s["out_q"]
    if op == "qk_norm_rope":
        be.qk_norm_rope(stream, t["q"], t["k"], t["qw"], t["kw"], EPS, t["positions"], s["rope"], out_q=t["out_q"],
                        out_k=t["out_k"])
        return [s["out_q"], s["out_k"]]
    if op == "paged_append":
        be.paged_append(stream, t["ck"], t["cv"], t["k"], t["v"], t["table"], t["positions"], seq_ids=t["seq_ids"],
                        rope=s["rope"])
        return s["ck"], s["cv"]
    be.paged_attention(stream, t["q"], t["ck"], t["cv"], t["table"], t["lens"], s["scale"],
                       query_starts=t.get("starts"), group_starts=t.get("group_starts"),
                       prefix_lens=t.get("prefix_lens"), out=t["out_q"])
    return s["out_q"]


def run(state):
    return _own(state) if own else _plain(state)


# --- 64 bits ----------------------------------------------------------------------------

def _exact_angles(c, positions):
    """[T, rotary / 2] angles and the factor, one pair after the other."""
    kind, theta, factor, orig = SCALINGS[c["scaling"]]
    d, out, scale = c["rotary"], [], 1.0
    for n in range(d // 2):
        f = math.exp(-2 * n / d * math.log(theta))
        if kind == "linear":
            f = f / factor
        elif kind == "bands":
            length = 2 * math.pi / f
            if length > orig / LOW_FREQ:
                f = f / factor
            elif length >= orig / HIGH_FREQ:
                smooth = (orig / length - LOW_FREQ) / (HIGH_FREQ - LOW_FREQ)
                f = (1 - smooth) * f / factor + smooth * f
        elif kind == "yarn":
            ends = [d / 2 * math.log(orig / (2 * math.pi * beta)) / math.log(theta) for beta in (BETA_FAST, BETA_SLOW)]
            low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), d - 1)
            share = min(1.0, max(0.0, (n - low) / max(high - low, 0.001)))
            f = f / factor * share + f * (1 - share)
            scale = 1.0 + 0.1 * math.log(factor)
        out.append(f)
    return positions.double()[:, None] * torch.tensor(out, dtype=torch.float64, device=positions.device), scale


def _exact_rotate(c, x, positions):
    angle, scale = _exact_angles(c, positions)
    turn = torch.polar(torch.full_like(angle, scale), angle)[:, None]
    y, d = x.clone(), c["rotary"]
    first, second = (slice(0, d // 2), slice(d // 2, d)) if c["layout"] == "half" else (slice(0, d, 2), slice(1, d, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "rope":
        return _exact_rotate(c, s["q"].double(), s["positions"])
    if c["op"] == "qk_norm_rope":
        out = []
        for x, w in ((s["q"].double(), s["qw"].double()), (s["k"].double(), s["kw"].double())):
            size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
            out.append(_exact_rotate(c, x * w / torch.sqrt(size ** 2 / c["dim"] + EPS), s["positions"]))
        return out
    if c["op"] == "paged_append":
        ck, cv = s["ck"].double(), s["cv"].double()
        flat = [x.view(-1, c["kv_heads"], c["dim"]) for x in (ck, cv)]
        pages = s["table"].index_select(0, s["seq_ids"]).gather(1, (s["positions"] // c["page"]).long()[:, None])[:, 0]
        rows = pages.long() * c["page"] + s["positions"] % c["page"]
        flat[0].index_copy_(0, rows, _exact_rotate(c, s["k"].double(), s["positions"]))
        flat[1].index_copy_(0, rows, s["v"].double())
        return ck, cv
    new, _, lens = _shape(c)
    out, first = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    share = c["heads"] // c["kv_heads"]
    for i, (n, length) in enumerate(zip(new, lens)):
        head = s["table"][i // c["seqs"] * c["seqs"]].long()
        tail = s["table"][i].long()
        slots = torch.arange(length, device="cuda")
        pages = torch.cat([head[slots[:c["prefix"]] // c["page"]], tail[slots[c["prefix"]:] // c["page"]]])
        k, v = (x[pages, slots % c["page"]].double() for x in (s["ck"], s["cv"]))
        q = s["q"][first:first + n].double()
        hidden = slots[None] > torch.arange(length - n, length, device="cuda")[:, None]
        for j in range(c["kv_heads"]):
            x = torch.einsum("thd,kd->htk", q[:, j * share:(j + 1) * share], k[:, j]) * s["scale"]
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[first:first + n, j * share:(j + 1) * share] = torch.einsum("htk,kd->thd", x, v[:, j])
        first += n
    return out
