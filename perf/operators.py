"""The serving operators of the kernel manager, as cases that can be timed and compared.

Three operators a decoder layer runs for a batch of sequences whose keys and values live in a
paged cache:

  append     rotates the new tokens' queries and keys by their positions and writes keys and
             values into the cache's pages
  attend     attention of the new tokens over the cache, for a batch whose sequences share
             their first positions (a system prompt), with a causal limit per token
  int4       products of a few tokens with a 4-bit weight matrix with group scales

`run` computes them with elementary torch operations in 32 bits (own = False), or through the
framework's entry points on raw device addresses (own = True).
"""
import math
import random

import torch

own = False

DT = {"f16": torch.float16, "f32": torch.float32}
SIZE = {"f16": 2, "f32": 4}


# ---------------------------------------------------------------------------- cases

def _append(name, **kw):
    c = dict(name=name, op="append", dtype="f16", heads=32, kv_heads=32, dim=128, page=16, seqs=1,
             new_min=1, new_max=1, past_max=0, rope="pairs", packed=False, ragged=1)
    c.update(kw)
    return c


def _attend(name, **kw):
    c = dict(name=name, op="attend", dtype="f16", heads=32, kv_heads=32, dim=128, page=16, seqs=1,
             new_min=1, new_max=1, shared=0, own_max=1, ragged=1)
    c.update(kw)
    return c


def _int4(name, **kw):
    c = dict(name=name, op="int4", dtype="f16", tokens=1, k=4096, n=4096, group=128, zeros=False)
    c.update(kw)
    return c


def listed():
    return [
        # one user's next token: nothing but latency
        _append("append 1 token", past_max=2000, ragged=3),
        # a serving batch of 64 sequences, grouped heads, q, k and v as one projection's output
        _append("append 64 tokens, grouped", kv_heads=8, seqs=64, past_max=3000, rope="halves",
                packed=True, ragged=5),
        # prompts of four users arriving together, 8 thousand tokens in all
        _append("append prompts", seqs=4, new_min=1500, new_max=2600, past_max=70, ragged=7),
        # one user's next token after a system prompt and a short conversation
        _attend("attend 1 token", shared=512, own_max=191, ragged=2),
        # 64 users of one long system prompt, grouped heads
        _attend("attend 64 tokens, long prefix", kv_heads=8, seqs=64, shared=8192, own_max=1024,
                ragged=4),
        # 32 users, a head of keys per head of queries (LLaMA-7B), odd lengths
        _attend("attend 32 tokens, 32 kv heads", seqs=32, shared=2043, own_max=701, ragged=6),
        # the rest of eight prompts behind a cached prefix, up to 256 new tokens each
        _attend("attend prompts", kv_heads=8, seqs=8, new_min=37, new_max=256, shared=2048,
                own_max=300, page=64, ragged=8),
        # the same path in 32 bits, small heads, a few speculated tokens per sequence
        _attend("attend f32", dtype="f32", heads=16, kv_heads=4, dim=64, seqs=19, new_min=1,
                new_max=5, shared=777, own_max=640, page=24, ragged=9),
        # a projection of one token (dim 4096)
        _int4("int4 1 token 4096x4096"),
        # the first feed-forward product of one token (4096 -> 11008)
        _int4("int4 1 token 4096x11008", n=11008),
        # the second one for a batch of 16 (11008 -> 4096), small groups with zero points
        _int4("int4 16 tokens 11008x4096", tokens=16, k=11008, n=4096, group=32, zeros=True),
        # the vocabulary's logits for five tokens, in 32 bits
        _int4("int4 f32 5 tokens 4096x32000", dtype="f32", tokens=5, n=32000, group=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "int4"])
    dtype = rng.choice(["f16", "f16", "f32"])
    ragged = rng.randrange(1 << 20)
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 32])
    dim = rng.choice([64, 80, 128, 128])
    page = rng.choice([8, 16, 24, 32, 64, 100])
    if op == "append":
        c = _append("", dtype=dtype, heads=heads, kv_heads=kv, dim=dim, page=page,
                    seqs=_log(rng, 1, 96), past_max=_log(rng, 1, 4000),
                    rope=rng.choice(["pairs", "halves"]), packed=rng.random() < 0.5, ragged=ragged)
        c["new_max"] = rng.choice([1, _log(rng, 1, max(1, 8000 // c["seqs"]))])
    elif op == "attend":
        c = _attend("", dtype=dtype, heads=heads, kv_heads=kv, dim=dim, page=page,
                    seqs=_log(rng, 1, 64), shared=rng.choice([0, _log(rng, 16, 8192)]),
                    ragged=ragged)
        c["own_max"] = _log(rng, 1, 1024)
        most = max(1, min(256, 2000 // c["seqs"], 16000000 // (heads * (c["shared"] + 1024))))
        c["new_max"] = min(c["own_max"], rng.choice([1, 1, _log(rng, 1, most)]))
    else:
        c = _int4("", dtype=dtype, tokens=_log(rng, 1, 32), k=32 * _log(rng, 16, 344),
                  n=_log(rng, 200, 20000), group=rng.choice([32, 64, 96, 128, 256]),
                  zeros=rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(c):
    """Per sequence: tokens new in this pass, and all of its tokens with those."""
    r = random.Random(c["ragged"])
    new = [r.randint(c["new_min"], c["new_max"]) for _ in range(c["seqs"])]
    if c["op"] == "append":
        return new, [n + r.randint(0, c["past_max"]) for n in new]
    return new, [c["shared"] + r.randint(n, max(n, c["own_max"])) for n in new]


def work(case):
    es = SIZE[case["dtype"]]
    if case["op"] == "int4":
        m, k, n = case["tokens"], case["k"], case["n"]
        groups = -(-k // case["group"])
        return {"bytes": n * k // 2 + n * groups * (es + (1 if case["zeros"] else 0)) +
                m * (k + n) * es, "flops": 2 * m * n * k}
    new, lens = _lengths(case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (h + 2 * kv) * d * es + tokens * d // 2 * 8,
                "flops": 3 * tokens * (h + kv) * d}
    seen = sum(n * ln - n * (n - 1) // 2 for n, ln in zip(new, lens))
    keys = case["shared"] + sum(ln - case["shared"] for ln in lens)
    return {"bytes": 2 * tokens * h * d * es + 2 * keys * kv * d * es, "flops": 4 * seen * h * d}


# ---------------------------------------------------------------------------- inputs

def _randn(gen, shape, dtype, sd=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * sd).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    dt = DT[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "int4":
        m, k, n, group = case["tokens"], case["k"], case["n"], case["group"]
        groups = -(-k // group)
        s["x"] = _randn(gen, (m, k), dt)
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda",
                               dtype=torch.uint8)
        s["scales"] = (0.002 + 0.004 * torch.rand((n, groups), generator=gen,
                                                  device="cuda")).to(dt)
        s["zeros"] = (torch.randint(4, 12, (n, groups), generator=gen, device="cuda",
                                    dtype=torch.uint8) if case["zeros"] else None)
        s["y"] = torch.empty((m, n), dtype=dt, device="cuda")
        return s
    new, lens = _lengths(case)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tokens, shared = sum(new), case.get("shared", 0)
    offs = [0]
    for n in new:
        offs.append(offs[-1] + n)
    # page tables: the pages that hold nothing but shared positions are one set for the whole
    # batch, the others are each sequence's own, in no order
    r = random.Random(case["ragged"] * 31 + int(seed))
    common = shared // page
    cols = max(1, max(-(-ln // page) for ln in lens))
    n_pages = common + sum(max(0, -(-ln // page) - common) for ln in lens) + 3
    ids = list(range(n_pages))
    r.shuffle(ids)
    rows, at = [], common
    for ln in lens:
        mine = max(0, -(-ln // page) - common)
        rows.append(ids[:common] + ids[at:at + mine] + [-1] * (cols - common - mine))
        at += mine
    s["offsets"], s["lens"], s["table"] = _ints(offs), _ints(lens), _ints(rows)
    s["k_cache"] = _randn(gen, (n_pages, page, kv, d), dt)
    s["v_cache"] = _randn(gen, (n_pages, page, kv, d), dt)
    tail = shared - common * page
    if tail:  # a page that is shared in part: each sequence has its copy of those positions
        mine = s["table"][:, common].long()
        for cache in (s["k_cache"], s["v_cache"]):
            cache[mine, :tail] = cache[mine[:1], :tail]
    s["n_pages"], s["tokens"] = n_pages, tokens
    if case["op"] == "attend":
        # queries of the size that a trained model's have: scores of a few units
        s["q"] = _randn(gen, (tokens, h, d), dt)
        s["out"] = torch.empty((tokens, h, d), dtype=dt, device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
        return s
    if case["packed"]:
        qkv = _randn(gen, (tokens, h + 2 * kv, d), dt)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    else:
        s["q"], s["k"], s["v"] = (_randn(gen, (tokens, x, d), dt) for x in (h, kv, kv))
    s["q_out"] = torch.empty((tokens, h, d), dtype=dt, device="cuda")
    n_pos = max(lens)
    ang = torch.outer(torch.arange(n_pos, dtype=torch.float64, device="cuda"),
                      10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d))
    s["freqs"] = torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()
    return s


# ---------------------------------------------------------------------------- the framework

_km = None


def _manager():
    global _km
    if _km is None:
        import einsummable_amd as ea

        _km = ea.KernelManager(0)
    return _km


def _call(s):
    """The call of one state as a function of the stream: descriptors are made once, as a
    program does that keeps its arena's addresses."""
    import einsummable_amd as ea

    c, km = s["case"], _manager()
    dt = {"f16": ea.F16, "f32": ea.F32}[c["dtype"]]
    if c["op"] == "int4":
        w = ea.Int4Weight(dt, c["n"], c["k"], c["group"], s["w"].data_ptr(),
                          s["scales"].data_ptr(), 0 if s["zeros"] is None else s["zeros"].data_ptr())
        y, x, m = s["y"].data_ptr(), s["x"].data_ptr(), c["tokens"]
        need = km.int4_linear_workspace(w, m)
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        ws = (s["workspace"].data_ptr(), need) if need else None
        return lambda stream: km.int4_linear(w, m, stream, y, x, ws)
    cache = ea.KvCache(dt, c["heads"], c["kv_heads"], c["dim"], s["n_pages"], c["page"],
                       s["k_cache"].data_ptr(), s["v_cache"].data_ptr())
    batch = ea.KvBatch(c["seqs"], s["tokens"], s["offsets"].data_ptr(), s["lens"].data_ptr(),
                       s["table"].data_ptr(), s["table"].shape[1])
    if c["op"] == "append":
        rope = {"pairs": ea.ROPE_PAIRS, "halves": ea.ROPE_HALVES}[c["rope"]]
        qo, q, k, v = (s[x].data_ptr() for x in ("q_out", "q", "k", "v"))
        fr, n_pos = s["freqs"].data_ptr(), s["freqs"].shape[0]
        strides = tuple(s[x].stride(0) for x in ("q_out", "q", "k", "v"))
        return lambda stream: km.kv_append(cache, batch, stream, qo, q, k, v, rope, fr, n_pos,
                                           strides)
    need = km.prefix_attention_workspace(cache, c["seqs"], s["tokens"], c["shared"])
    s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    ws = (s["workspace"].data_ptr(), need) if need else None
    out, q, shared, scale = s["out"].data_ptr(), s["q"].data_ptr(), c["shared"], s["scale"]
    return lambda stream: km.prefix_attention(cache, batch, shared, scale, stream, out, q, ws)


# ---------------------------------------------------------------------------- plain forms

def _tokens(s):
    """Sequence and position of every token."""
    t = torch.arange(s["tokens"], device="cuda")
    offs = s["offsets"].long()
    seq = torch.bucketize(t, offs[1:], right=True)
    return seq, s["lens"].long()[seq] - offs[seq + 1] + t


def _rotate(x, cs, rope):
    x = x.float()
    if rope == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, dim=-1)
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    re, im = a * c - b * sn, a * sn + b * c
    return torch.stack([re, im], dim=-1).flatten(-2) if rope == "pairs" else torch.cat([re, im], -1)


def _plain_append(s):
    c = s["case"]
    seq, pos = _tokens(s)
    page = s["table"].long()[seq, pos // c["page"]]
    cs = s["freqs"][pos]
    s["q_out"].copy_(_rotate(s["q"], cs, c["rope"]))
    s["k_cache"][page, pos % c["page"]] = _rotate(s["k"], cs, c["rope"]).to(s["k_cache"].dtype)
    s["v_cache"][page, pos % c["page"]] = s["v"]
    return s["q_out"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    c = s["case"]
    kv, d, page, shared, b = c["kv_heads"], c["dim"], c["page"], c["shared"], c["seqs"]
    g = c["heads"] // kv
    seq, pos = _tokens(s)
    row = torch.arange(s["tokens"], device="cuda") - s["offsets"].long()[seq]
    n = c["new_max"]
    # the tokens as [sequence, kv head, token and head of its group, dim]; rows of tokens that
    # a sequence does not have are computed and dropped
    q = torch.zeros((b, n, kv, g, d), dtype=torch.float32, device="cuda")
    q[seq, row] = s["q"].float().view(-1, kv, g, d)
    q = (q * s["scale"]).permute(0, 2, 1, 3, 4).reshape(b, kv, n * g, d)
    limit = torch.full((b, n), -1, dtype=torch.long, device="cuda")
    limit[seq, row] = pos
    table = s["table"].long()

    def rows_of(t, at):
        where = t[..., at // page].clamp_min(0), at % page
        return [x[where].float() for x in (s["k_cache"], s["v_cache"])]

    p0 = torch.arange(shared, device="cuda")
    p1 = torch.arange(shared, table.shape[1] * page, device="cuda")
    k0, v0 = rows_of(table[0], p0)                                    # [shared, kv, d]
    k1, v1 = rows_of(table, p1)                                       # [b, rest, kv, d]
    k0, v0 = (x.permute(1, 0, 2).contiguous() for x in (k0, v0))
    k1, v1 = (x.permute(0, 2, 1, 3).contiguous() for x in (k1, v1))
    q0 = q.transpose(0, 1).reshape(kv, b * n * g, d)
    s0 = (q0 @ k0.transpose(1, 2)).view(kv, b, n * g, shared).transpose(0, 1)
    sc = torch.cat([s0, q @ k1.transpose(2, 3)], dim=-1)              # [b, kv, n g, positions]
    seen = torch.cat([p0, p1]) <= limit.repeat_interleave(g, dim=1)[:, None, :, None]
    sc = sc.masked_fill(~seen, -math.inf)
    sc = torch.exp(sc - sc.amax(dim=-1, keepdim=True).clamp_min(-1e30))
    total = sc.sum(dim=-1, keepdim=True)
    w0 = sc[..., :shared].transpose(0, 1).reshape(kv, b * n * g, shared)
    o = (w0 @ v0).view(kv, b, n * g, d).transpose(0, 1) + sc[..., shared:] @ v1
    o = (o / total).view(b, kv, n, g, d).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o[seq, row].reshape(-1, c["heads"], d))
    return s["out"]


def _plain_int4(s):
    c = s["case"]
    q = torch.stack([s["w"] & 15, s["w"] >> 4], dim=-1).flatten(1).float()
    of = torch.arange(c["k"], device="cuda") // c["group"]
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, of]
    w = (q - zero) * s["scales"].float()[:, of]
    s["y"].copy_(s["x"].float() @ w.t())
    return s["y"]


def run(state):
    op = state["case"]["op"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        state["call"](torch.cuda.current_stream().cuda_stream)
        if op == "append":
            return state["q_out"], state["k_cache"], state["v_cache"]
        return state["out"] if op == "attend" else state["y"]
    if op == "append":
        return _plain_append(state)
    return _plain_attend(state) if op == "attend" else _plain_int4(state)


# ---------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int4":
        x = s["x"].double()
        y = torch.empty((case["tokens"], case["n"]), dtype=torch.float64, device="cuda")
        for lo in range(0, case["n"], 2048):          # a strip of the weight at a time
            w = s["w"][lo:lo + 2048].long()
            full = torch.zeros((w.shape[0], case["k"]), dtype=torch.float64, device="cuda")
            full[:, 0::2], full[:, 1::2] = (w % 16).double(), (w // 16).double()
            for gi in range(s["scales"].shape[1]):
                cols = slice(gi * case["group"], (gi + 1) * case["group"])
                z = 8.0 if s["zeros"] is None else s["zeros"][lo:lo + 2048, gi:gi + 1].double()
                full[:, cols] = (full[:, cols] - z) * s["scales"][lo:lo + 2048, gi:gi + 1].double()
            y[:, lo:lo + 2048] = x @ full.t()
        return y
    new, lens = _lengths(case)
    d, page, g = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    at = 0
    if case["op"] == "append":
        qo = torch.empty(s["q_out"].shape, dtype=torch.float64, device="cuda")
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b, (n, ln) in enumerate(zip(new, lens)):
            pos = torch.arange(ln - n, ln, device="cuda")
            turn = torch.view_as_complex(s["freqs"][ln - n:ln].double()).unsqueeze(1)

            def turned(x):
                x = x[at:at + n].double()
                if case["rope"] == "halves":
                    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn
                    return torch.cat([z.real, z.imag], dim=-1)
                z = torch.complex(x[..., 0::2], x[..., 1::2]) * turn
                return torch.view_as_real(z).reshape(x.shape)

            pages = s["table"][b].long()[pos // page]
            qo[at:at + n] = turned(s["q"])
            kc[pages, pos % page] = turned(s["k"])
            vc[pages, pos % page] = s["v"][at:at + n].double()
            at += n
        return qo, kc, vc
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    for b, (n, ln) in enumerate(zip(new, lens)):
        pos = torch.arange(ln, device="cuda")
        pages = s["table"][b].long()[pos // page]
        k, v = (x[pages, pos % page].double().repeat_interleave(g, dim=1).transpose(0, 1)
                .contiguous() for x in (s["k_cache"], s["v_cache"]))  # [heads, positions, d]
        q = s["q"][at:at + n].double().transpose(0, 1).contiguous()
        sc = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        last = torch.arange(ln - n, ln, device="cuda")
        sc = torch.where(pos[None, :] <= last[:, None], sc, -math.inf)
        out[at:at + n] = torch.matmul(torch.softmax(sc, dim=-1), v).transpose(0, 1)
        at += n
    return out
