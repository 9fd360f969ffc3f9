"""The operators of a paged KV cache, as cases that can be timed and whose outputs can be compared.

Three kinds of case, each one call of `paged`:

  append   the projected queries, keys and values of a step's tokens: queries and keys rotated to their positions, keys and
           values stored in the pages of their sequences
  attend   attention of a batch of sequences over their pages: single tokens, drafted tokens, prompts, and all of them together
  prefix   the same for a batch that shares the pages of a long prefix

A case's sequence lengths come from the case alone (`mix`), so that its work is known without its inputs. Where `own` is false,
`run` computes the plain form: gathers, products, exponentials and sums of torch in 32 bits (angles in 64).
"""
import importlib
import math
import random
import struct
import types

import torch

own = False


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    layer8 = {"heads": 32, "kv_heads": 8, "D": 128}          # an 8B-sized layer with grouped KV heads
    small = {"heads": 14, "kv_heads": 2, "D": 64}            # a small model whose group of 7 divides no tile
    rope = {"n_dims": 128, "neox": False, "base": 500000.0, "yarn": False, "factors": False, "far": 0, "pad": 0}
    plain = {"window": 0, "softcap": 0.0}
    return [
        # one user, one new token: launch and latency
        {"name": "append_1", "kind": "append", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 700, "kv_hi": 700, "page": 16, "layout": "token",
         "mix": 1, **layer8, **rope},
        # a serving step of a padded batch: partial NEOX rotation with frequency factors, positions far out
        {"name": "append_padded_200", "kind": "append", "seqs": 200, "q_lo": 0, "q_hi": 2, "kv_lo": 1, "kv_hi": 900, "page": 32, "layout": "head",
         "mix": 2, "heads": 20, "kv_heads": 5, "D": 128, **{**rope, "n_dims": 96, "neox": True, "factors": True, "far": 300000, "pad": 56}},
        # prompts of a batch, stretched context
        {"name": "append_prompts_8k", "kind": "append", "seqs": 5, "q_lo": 777, "q_hi": 2048, "kv_lo": 777, "kv_hi": 2048, "page": 16,
         "layout": "token", "mix": 3, **layer8, **{**rope, "yarn": True}},
        # one user, a short context: latency
        {"name": "attend_1x500", "kind": "attend", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 500, "kv_hi": 500, "page": 16, "layout": "token",
         "out": "f32", "mix": 4, **layer8, **plain},
        # one user, a whole book in the context
        {"name": "attend_1x131072", "kind": "attend", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 131072, "kv_hi": 131072, "page": 64,
         "layout": "head", "out": "f32", "mix": 5, **layer8, **plain},
        # a serving step: users at very different places in their contexts
        {"name": "attend_ragged_96", "kind": "attend", "seqs": 96, "q_lo": 1, "q_hi": 1, "kv_lo": 20, "kv_hi": 8192, "page": 16, "layout": "token",
         "out": "f16", "mix": 6, **layer8, **plain},
        # drafted tokens of a small model under a sliding window
        {"name": "attend_draft_32", "kind": "attend", "seqs": 32, "q_lo": 1, "q_hi": 6, "kv_lo": 100, "kv_hi": 3000, "page": 32, "layout": "token",
         "out": "f16", "mix": 7, **small, "window": 1024, "softcap": 30.0},
        # a chunk of one prompt beside the tokens of the others (chunked prefill); results for a 32-bit consumer
        {"name": "attend_mixed_24", "kind": "attend", "seqs": 24, "q_lo": 1, "q_hi": 512, "kv_lo": 200, "kv_hi": 2500, "page": 16,
         "layout": "token", "out": "f32", "mix": 8, **layer8, **plain},
        # the largest: a whole prompt at once
        {"name": "attend_prompt_8192", "kind": "attend", "seqs": 1, "q_lo": 8192, "q_hi": 8192, "kv_lo": 8192, "kv_hi": 8192, "page": 64,
         "layout": "head", "out": "f16", "mix": 9, **layer8, **plain},
        # a few users behind one system prompt, short answers so far: latency
        {"name": "prefix_6x1000", "kind": "prefix", "seqs": 6, "q_lo": 1, "q_hi": 1, "kv_lo": 1, "kv_hi": 90, "prefix": 1000, "page": 16,
         "layout": "token", "out": "f32", "mix": 10, **layer8, "softcap": 0.0},
        # many samples of one long question
        {"name": "prefix_64x8192", "kind": "prefix", "seqs": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 30, "kv_hi": 1000, "prefix": 8192, "page": 16,
         "layout": "token", "out": "f16", "mix": 11, **layer8, "softcap": 0.0},
        # new questions of several tokens about one document
        {"name": "prefix_160x30001", "kind": "prefix", "seqs": 160, "q_lo": 1, "q_hi": 12, "kv_lo": 1, "kv_hi": 300, "prefix": 30001, "page": 64,
         "layout": "head", "out": "f16", "mix": 12, **layer8, "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    D = rng.choice([64, 128, 128])
    kv_heads, group = rng.randint(1, 10), rng.randint(1, 8)
    return {"heads": kv_heads * group, "kv_heads": kv_heads, "D": D}


def draw(rng):
    c = {"kind": rng.choice(["append", "attend", "attend", "attend", "prefix"]), **_heads(rng), "page": rng.choice([16, 32, 64, 128]),
         "layout": rng.choice(["token", "head"]), "mix": rng.randrange(1 << 20)}
    if c["kind"] == "append":
        tokens = _log(rng, 1, 8192)
        c["seqs"] = _log(rng, 1, min(tokens, 256))
        c["q_hi"] = max(1, tokens // c["seqs"])
        c["q_lo"] = rng.choice([0, 1, c["q_hi"] // 2, c["q_hi"]])
        c["kv_lo"], c["kv_hi"] = max(1, c["q_lo"]), c["q_hi"] + rng.choice([0, _log(rng, 1, 500)])
        c |= {"n_dims": rng.choice([c["D"], c["D"], c["D"] // 2, 2 * rng.randint(1, c["D"] // 2)]), "neox": rng.random() < 0.5,
              "base": rng.choice([10000.0, 500000.0]), "yarn": rng.random() < 0.3, "factors": rng.random() < 0.3,
              "far": rng.choice([0, 0, _log(rng, 1000, 1000000)]), "pad": rng.choice([0, rng.randint(1, 64)])}
        return c
    c |= {"softcap": rng.choice([0.0, 0.0, 30.0]), "out": rng.choice(["f16", "f32"])}
    if c["kind"] == "prefix":
        c["prefix"] = _log(rng, 200, 32768)
        c["seqs"], c["q_hi"] = _log(rng, 2, 192), rng.choice([1, 1, rng.randint(2, 12)])
        c["q_lo"] = rng.choice([0, 1]) if c["q_hi"] > 1 else 1
        c["kv_lo"], c["kv_hi"] = 1, max(c["q_hi"], _log(rng, 1, 1000))
        while c["seqs"] * c["q_hi"] * c["heads"] * c["prefix"] > 1 << 30:
            c["prefix"] = c["prefix"] // 2 + 1
        return c
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    form = rng.choice(["token", "token", "draft", "prompt", "mixed"])
    c["seqs"] = {"token": _log(rng, 1, 256), "draft": _log(rng, 1, 64), "prompt": _log(rng, 1, 6), "mixed": _log(rng, 2, 32)}[form]
    c["q_hi"] = {"token": 1, "draft": rng.randint(2, 16), "prompt": _log(rng, 17, 8192), "mixed": _log(rng, 17, 700)}[form]
    c["q_lo"] = {"token": 1, "draft": rng.randint(0, 2), "prompt": c["q_hi"] // 3, "mixed": 1}[form]
    c["kv_hi"] = _log(rng, 16, 131072)
    while c["seqs"] * c["kv_hi"] * c["kv_heads"] * c["D"] > 1 << 29 or c["seqs"] * c["q_hi"] * c["kv_hi"] * c["heads"] > 1 << 30:
        c["kv_hi"] = c["kv_hi"] // 2 + 1
    c["kv_hi"] = max(c["q_hi"], c["kv_hi"])
    while c["seqs"] * c["q_hi"] * c["kv_hi"] * c["heads"] > 1 << 31:   # (a prompt longer than what was left for its keys)
        c["q_hi"], c["q_lo"] = c["q_hi"] // 2 + 1, c["q_lo"] // 2
        c["kv_hi"] = c["q_hi"]
    c["kv_lo"] = rng.choice([1, c["kv_hi"] // 2 + 1, c["kv_hi"]])
    return c


def _lengths(c):
    """New tokens and keys (the new ones among them) of every sequence: lengths spread over their logarithm, the largest taken."""
    rng = random.Random(c["mix"])
    n = []
    for i in range(c["seqs"]):
        q = c["q_hi"] if i == 0 else rng.randint(c["q_lo"], c["q_hi"]) if c["q_hi"] <= 16 or c["q_lo"] > 1 else c["q_lo"]
        n.append((q, max(q, c["kv_hi"] if i == 0 else _log(rng, c["kv_lo"], c["kv_hi"]))))
    rng.shuffle(n)
    return [a for a, _ in n], [b for _, b in n]


def work(case):
    qs, kvs = _lengths(case)
    H, Hkv, D = case["heads"], case["kv_heads"], case["D"]
    rows = sum(qs)
    if case["kind"] == "append":
        return {"bytes": rows * (H + 2 * Hkv) * D * 6, "flops": 3 * rows * (H + Hkv) * D}
    w = case.get("window") or 1 << 40
    pairs = keys = 0
    for q, kv in zip(qs, kvs):
        if q:
            keys += min(kv, w + q - 1)
            # (query, key) pairs under the causal limit and the window
            pairs += sum(min(kv - q + j + 1, w) for j in range(q)) if q < 64 or w < 1 << 40 else q * (kv - q) + q * (q + 1) // 2
    pairs += rows * case.get("prefix", 0)
    keys += case.get("prefix", 0)
    return {"bytes": 4 * keys * Hkv * D + rows * H * D * (2 + (2 if case["out"] == "f16" else 4)), "flops": 4 * pairs * H * D}


# ---- what a program has in hand ----------------------------------------------------------------------------------------
def _theta_scale(c):
    """The factor between the angles of neighbouring pairs, the 32-bit number that the rotation is given."""
    return struct.unpack("<f", struct.pack("<f", c["base"] ** (-2.0 / c["n_dims"])))[0]


def _yarn(c):
    """freq_scale, ext_factor, attn_factor and the two pairs between which YaRN blends."""
    return (0.25, 1.0, 1.0, 0.2 * c["n_dims"], 0.4 * c["n_dims"]) if c["yarn"] else (1.0, 0.0, 1.0, 0.0, 0.0)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = types.SimpleNamespace(case=c, plan=None)
    qs, kvs = _lengths(c)
    S, P, Hkv, H, D = c["seqs"], c["page"], c["kv_heads"], c["heads"], c["D"]
    s.rows = sum(qs)                                        # tokens of the batch
    s.held = s.rows + c.get("pad", 0)                       # rows of its tensors
    s.max_q, s.max_kv = max(qs), max(kvs)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s.q_start = ints([sum(qs[:i]) for i in range(S + 1)])
    s.kv_len = ints(kvs)
    need = [(n + P - 1) // P for n in kvs]
    prefix_pages = (c.get("prefix", 0) + P - 1) // P
    s.n_pages = sum(need) + prefix_pages + 3
    pages = torch.randperm(s.n_pages, device="cuda", generator=gen).to(torch.int32)    # the pool hands pages out in any order
    s.width = max(need)
    first = torch.tensor([sum(need[:i]) for i in range(S)], device="cuda").view(-1, 1)
    column = torch.arange(s.width, device="cuda").view(1, -1)
    held = column < ints(need).view(-1, 1)
    s.table = torch.where(held, pages[(first + column).clamp(max=s.n_pages - 1)], 0).contiguous()   # behind a sequence's last page: anything
    s.prefix = torch.cat([ints([c.get("prefix", 0)]), pages[sum(need):sum(need) + prefix_pages]]) if prefix_pages else None
    shape = (s.n_pages, P, Hkv, D) if c["layout"] == "token" else (s.n_pages, Hkv, P, D)
    s.k_cache, s.v_cache = normal(*shape).half(), normal(*shape).half()
    if c["kind"] == "append":
        s.q, s.k, s.v = normal(s.held, H, D), normal(s.held, Hkv, D), normal(s.held, Hkv, D)
        s.q_out = torch.full((s.held, H, D), 0.5, dtype=torch.float16, device="cuda")
        s.factors = torch.rand(c["n_dims"] // 2, device="cuda", generator=gen) * 7.0 + 1.0 if c["factors"] else None
        at, _, place = _places(s)
        s.positions = None
        if c["far"]:
            s.positions = torch.full((s.held,), -1, dtype=torch.int32, device="cuda")
            s.positions[:s.rows] = (place + c["far"]).to(torch.int32)
    else:
        s.q = normal(s.held, H, D).half()
        s.dst = torch.full((s.held, H, D), 0.015625, dtype=torch.float16 if c["out"] == "f16" else torch.float32, device="cuda")
    return s


def _places(s):
    """Of every token: its sequence, its number among the sequence's new tokens, its place among the sequence's keys."""
    token = torch.arange(s.rows, device="cuda")
    seq = torch.bucketize(token, s.q_start[1:].long(), right=True)
    j = token - s.q_start[seq]
    n = s.q_start[seq + 1] - s.q_start[seq]
    return seq, j, s.kv_len[seq] - n + j


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _angles(c, positions, factors):
    """cosine and sine, times the magnitude, of every (position, pair), from angles in 64 bits."""
    pair = torch.arange(c["n_dims"] // 2, device="cuda", dtype=torch.float64)
    scale, ext, magnitude, low, high = _yarn(c)
    far = positions.double().view(-1, 1) * _theta_scale(c) ** pair
    if factors is not None:
        far = far / factors.double()
    angle = far * scale
    if ext:
        ramp = (1.0 - ((pair - low) / max(0.001, high - low)).clamp(0.0, 1.0)) * ext
        angle = angle * (1.0 - ramp) + far * ramp
        magnitude = magnitude * (1.0 + 0.1 * math.log(1.0 / scale))
    return torch.cos(angle) * magnitude, torch.sin(angle) * magnitude


def _rotate(c, x, cos, sin):
    n = c["n_dims"]
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if c["neox"] else (x[..., 0:n:2], x[..., 1:n:2])
    cos, sin = cos.to(x.dtype).unsqueeze(1), sin.to(x.dtype).unsqueeze(1)
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([y0, y1], -1) if c["neox"] else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., n:]], -1)


def _append_plain(s):
    c, n, P = s.case, s.rows, s.case["page"]
    seq, _, place = _places(s)
    cos, sin = _angles(c, place if s.positions is None else s.positions[:n], s.factors)
    s.q_out[:n] = _rotate(c, s.q[:n], cos, sin).half()
    page, token = s.table[seq, place // P].long(), place % P
    for cache, x in ((s.k_cache, _rotate(c, s.k[:n], cos, sin)), (s.v_cache, s.v[:n])):
        if c["layout"] == "token":
            cache[page, token] = x.half()
        else:
            cache[page, :, token] = x.half()
    return [s.q_out, s.k_cache, s.v_cache]


def _pages(s, cache, table):
    """[..., kv_heads, keys, D] in 32 bits of the pages of a table [..., pages]."""
    x = cache[table.long()].float()                                  # [..., pages, token, head, D] or [..., pages, head, token, D]
    x = x.transpose(-2, -3) if s.case["layout"] == "token" else x
    return x.transpose(-3, -4).flatten(-3, -2)


def _part(s, q, k, v, seen):
    """Maximum, sum and weighted values of one set of keys: q [..., rows, D], k and v [..., keys, D], seen: which keys a row sees."""
    c = s.case
    x = (q @ k.transpose(-1, -2)) * c["D"] ** -0.5
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    if seen is not None:
        x = torch.where(seen, x, float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    return m, p.sum(-1, keepdim=True), p @ v


def _attend_plain(s):
    c, n = s.case, s.rows
    H, Hkv, D, G, S, Q = c["heads"], c["kv_heads"], c["D"], c["heads"] // c["kv_heads"], c["seqs"], s.max_q
    seq, j, _ = _places(s)
    q = s.q[:n].float().view(n, Hkv, G, D)
    padded = torch.zeros((S, Q, Hkv, G, D), device="cuda")
    padded[seq, j] = q
    padded = padded.permute(0, 2, 1, 3, 4).reshape(S, Hkv, Q * G, D)
    k, v = _pages(s, s.k_cache, s.table), _pages(s, s.v_cache, s.table)
    key = torch.arange(k.shape[-2], device="cuda")
    last = (s.kv_len - (s.q_start[1:] - s.q_start[:-1])).view(S, 1) + torch.arange(Q, device="cuda")     # the key at a query's own place
    seen = (key <= last.unsqueeze(-1)) & (key < s.kv_len.view(S, 1, 1))
    if c.get("window"):
        seen &= key > (last - c["window"]).unsqueeze(-1)
    m, l, o = _part(s, padded, k, v, seen.repeat_interleave(G, 1).unsqueeze(1))
    m, l, o = (x.view(S, Hkv, Q, G, -1).transpose(1, 2)[seq, j] for x in (m, l, o))      # [rows, Hkv, G, ...]
    if c["kind"] == "prefix":
        kp, vp = _pages(s, s.k_cache, s.prefix[1:])[:, :c["prefix"]], _pages(s, s.v_cache, s.prefix[1:])[:, :c["prefix"]]
        m2, l2, o2 = (x.view(Hkv, n, G, -1).transpose(0, 1) for x in _part(s, q.transpose(0, 1).reshape(Hkv, n * G, D), kp, vp, None))
        top = torch.maximum(m, m2)
        a, b = torch.exp(m - top), torch.exp(m2 - top)
        l, o = l * a + l2 * b, o * a + o2 * b
    s.dst[:n] = torch.where(l > 0, o / l, 0.0).reshape(n, H, D).to(s.dst.dtype)
    return s.dst


# ---- the framework's calls ---------------------------------------------------------------------------------------------
_context = _stream = None


class _Plan:
    """A call recorded once and replayed, as a serving loop does it; what it created is destroyed with it. The context's stream and torch's
    know nothing of one another, so the program makes the context's stream torch's, too: a pass is ordered behind what torch has made of its
    inputs, and torch behind the pass, without events (5 us a pass of host time)."""

    def __init__(self, s):
        global _context, _stream
        amv = importlib.import_module("ameva-compute_b200")
        if _context is None:
            _context = amv.runtime.init()
            _stream = torch.cuda.ExternalStream(_context.stream)
        _stream.wait_stream(torch.cuda.current_stream())      # (the inputs were made there)
        torch.cuda.set_stream(_stream)
        paged, ctx, c = amv.paged, _context, s.case
        self.owned, self.tensors, self.event = [], [], None

        def bind(t):
            self.tensors.append(t)
            self.owned.append(ctx.import_buffer(t.data_ptr(), t.numel() * t.element_size()))
            return self.owned[-1]

        status = bind(torch.tensor([0, -1], dtype=torch.int32, device="cuda"))
        cache = paged.Cache(bind(s.k_cache), bind(s.v_cache), s.n_pages, c["page"], c["kv_heads"], c["D"], layout=c["layout"])
        seqs = paged.Sequences(bind(s.table), bind(s.q_start), bind(s.kv_len), n_seqs=c["seqs"], table_stride=s.width, rows=s.held,
                               max_q=s.max_q, max_kv=s.max_kv)
        self.batch = ctx.batch(4)
        if c["kind"] == "append":
            scale, ext, attn, low, high = _yarn(c)
            rope = paged.Rope(c["n_dims"], _theta_scale(c), neox=c["neox"], freq_scale=scale, ext_factor=ext, attn_factor=attn, corr=(low, high))
            paged.record_append(self.batch, cache, seqs, bind(s.q), bind(s.k), bind(s.v), bind(s.q_out), status, heads=c["heads"], rope=rope,
                                positions=None if s.positions is None else bind(s.positions),
                                factors=None if s.factors is None else bind(s.factors))
            self.out = [s.q_out, s.k_cache, s.v_cache]
        else:
            prefix = s.prefix is not None
            scratch = ctx.buffer(paged.scratch_bytes(ctx, seqs, heads=c["heads"], head_dim=c["D"], prefix=prefix))
            self.owned.append(scratch)
            more = {"prefix": bind(s.prefix), "max_prefix": c["prefix"]} if prefix else {"window": c["window"]}
            (paged.record_prefix_attention if prefix else paged.record_attention)(
                self.batch, cache, seqs, bind(s.q), bind(s.dst), scratch, status, heads=c["heads"], scale=c["D"] ** -0.5,
                softcap=c["softcap"], f16_out=c["out"] == "f16", **more)
            self.out = s.dst
        self.batch.instantiate()

    def run(self):
        if self.event is not None:
            self.event.destroy()      # of the pass before
        self.event = self.batch.replay()
        return self.out

    def __del__(self):
        try:
            if self.event is not None:
                self.event.destroy()
            self.batch.destroy()
            for b in reversed(self.owned):
                b.destroy()
        except Exception:
            pass


def run(state):
    if own:
        if state.plan is None:
            state.plan = _Plan(state)
        return state.plan.run()
    return _append_plain(state) if state.case["kind"] == "append" else _attend_plain(state)


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    qs, kvs = _lengths(c)
    P, H, Hkv, D = c["page"], c["heads"], c["kv_heads"], c["D"]
    G = H // Hkv
    if c["kind"] == "append":
        out = [t.double() for t in (s.q_out, s.k_cache, s.v_cache)]
        n, half = c["n_dims"], c["n_dims"] // 2
        scale, ext, magnitude, low, high = _yarn(c)
        if ext:
            magnitude *= 1 + 0.1 * math.log(1 / scale)
        row = 0
        for i, (q, kv) in enumerate(zip(qs, kvs)):
            if not q:
                continue
            place = torch.arange(kv - q, kv, device="cuda")
            at = place.double() + c["far"]
            pair = torch.arange(half, dtype=torch.float64, device="cuda")
            full = torch.outer(at, torch.exp(pair * math.log(_theta_scale(c))) / (1.0 if s.factors is None else s.factors.double()))
            share = torch.clip(1 - torch.clip((pair - low) / max(0.001, high - low), 0, 1), 0, 1) * ext
            angle = full * scale * (1 - share) + full * share
            turn = torch.polar(torch.full_like(angle, magnitude), angle).unsqueeze(1)      # e^(i angle) of every pair
            first, second = (slice(0, half), slice(half, n)) if c["neox"] else (slice(0, n, 2), slice(1, n, 2))
            turned = [s.q[row:row + q].double(), s.k[row:row + q].double()]
            for y in turned:
                z = torch.complex(y[:, :, first], y[:, :, second]) * turn
                y[:, :, first], y[:, :, second] = z.real, z.imag
            out[0][row:row + q], k = turned
            v = s.v[row:row + q].double()
            page = s.table[i].long()[place // P]
            if c["layout"] == "token":
                out[1][page, place % P], out[2][page, place % P] = k, v
            else:
                out[1][page, :, place % P], out[2][page, :, place % P] = k, v
            row += q
        return out
    out = s.dst.double()

    def keys(cache, pages, n, h):
        x = cache[pages.long(), :, h] if c["layout"] == "token" else cache[pages.long(), h]
        return x.reshape(-1, D)[:n].double()

    row = 0
    for i, (q, kv) in enumerate(zip(qs, kvs)):
        if not q:
            continue
        for h in range(Hkv):
            k, v = keys(s.k_cache, s.table[i], kv, h), keys(s.v_cache, s.table[i], kv, h)
            place = torch.arange(kv - q, kv, device="cuda").view(-1, 1)
            key = torch.arange(kv, device="cuda").view(1, -1)
            hidden = (key > place) | (key <= place - (c.get("window") or 1 << 40))
            if c["kind"] == "prefix":
                if row == 0 and h == 0:
                    shared = [(keys(s.k_cache, s.prefix[1:], c["prefix"], g), keys(s.v_cache, s.prefix[1:], c["prefix"], g)) for g in range(Hkv)]
                k, v = torch.cat([shared[h][0], k]), torch.cat([shared[h][1], v])
                hidden = torch.cat([torch.zeros((q, c["prefix"]), dtype=torch.bool, device="cuda"), hidden], 1)
            for g in range(h * G, h * G + G):
                x = s.q[row:row + q, g].double() @ k.T / math.sqrt(D)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                out[row:row + q, g] = torch.softmax(x.masked_fill(hidden, float("-inf")), 1) @ v
        row += q
    return out
