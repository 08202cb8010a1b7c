"""What the paged-cache and prompt operators do, in plain torch and through the framework, and the cases they are
measured on.

A case is one pass of one step of serving several sequences whose keys and values lie in pages:

  append   new tokens' queries and keys are (normalised and) rotated, keys and values stored in fp16 pages
  extend   the same into 4-bit pages, then the sequences' whole context read back as fp16 (a prompt continued)
  read     cached keys and values read back as fp16
  prefill  causal attention of packed prompts (or of prompt chunks over a longer context)
  decode   one query per sequence over its pages, fp16 or 4 bits

Page layouts (page = positions per page, hd = head_dim):

  fp16     [pages, kv heads, page, hd]
  4 bits   K uint8 [pages, kv heads, page, hd/2 + hd/16]: a block of page * hd/2 bytes of codes, then page * hd/32
           fp16 scales (one per 32 values).  A position's codes are hd/8 little-endian words; word t * (hd/32) + j
           holds values 32 j + 8 t + (0..7), value 2 i in nibble i and 2 i + 1 in nibble i + 4.
           V uint8 [pages, kv heads, page, hd/2 + 2]: page * hd/2 bytes of codes, then page fp16 scales (one per
           position).  Positions 2 m and 2 m + 1 share hd/4 words; word w holds values 4 w + (0..3), the even
           position's in nibbles 0..3, the odd one's in nibbles 4..7.
           Codes are two's-complement nibbles in [-7, 7]; a value is code * scale.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
GROUP = 32  # values of a key that share a scale


def _ops():
    """The framework's operators, imported once as a program does."""
    if "soinfer.ops" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "sparse-offload-infer_b200"))
        import soinfer.ops  # noqa: F401
    return sys.modules["soinfer.ops"]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of one sequence enters the cache: a launch's latency
        dict(name="append-one", op="append", bits=16, nq=16, nkv=8, hd=128, page=16, new="1", past="777", norm=True),
        # five prompts of a batch prefilled at once, q / k / v as slices of one projection's output
        dict(name="append-prompts", op="append", bits=16, nq=40, nkv=8, hd=128, page=64, new="4096,1,2501,777,1300",
             past="0,0,0,0,0", norm=True),
        # three prompt chunks join 4-bit caches; the chunk attention needs the whole context in fp16
        dict(name="extend-int4", op="extend", bits=4, nq=16, nkv=8, hd=128, page=32, new="2048,511,1200",
             past="8192,333,4001", norm=True),
        # a long cached document handed to the next prompt chunk
        dict(name="read-int4-long", op="read", bits=4, nq=8, nkv=8, hd=128, page=64, past="65431"),
        # two cached contexts of a small-head model
        dict(name="read-f16", op="read", bits=16, nq=4, nkv=4, hd=64, page=16, past="2047,3001"),
        # a short question: latency
        dict(name="prefill-short", op="prefill", nq=16, nkv=8, hd=128, new="37", past="0"),
        # a batch of unequal prompts
        dict(name="prefill-packed", op="prefill", nq=16, nkv=8, hd=128, new="1500,129,64,1,777,1024,333",
             past="0,0,0,0,0,0,0"),
        # one long prompt of the 40-head configuration
        dict(name="prefill-long", op="prefill", nq=40, nkv=8, hd=128, new="8192", past="0"),
        # chunks of two prompts over their cached contexts, 64-wide heads
        dict(name="prefill-chunk-hd64", op="prefill", nq=32, nkv=4, hd=64, new="512,1000", past="3500,2047"),
        # one chat, one token: latency
        dict(name="decode-int4-one", op="decode", bits=4, nq=16, nkv=8, hd=128, page=16, past="777"),
        # two very long documents, 40-head configuration
        dict(name="decode-int4-long", op="decode", bits=4, nq=40, nkv=8, hd=128, page=64, past="131072,100003"),
        # a full batch of unequal chats, fp16 pages
        dict(name="decode-f16-batch", op="decode", bits=16, nq=32, nkv=4, hd=128, page=32,
             past="4096,3000,17,1999,2500,1023,4001,640"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lengths(rng, total, most):
    n = rng.randint(1, most)
    cut = [rng.random() + 0.05 for _ in range(n)]
    return [max(1, int(total * c / sum(cut))) for c in cut]


def draw(rng):
    op = rng.choice(["append", "extend", "read", "prefill", "decode", "decode"])
    nq, nkv, hd = rng.choice([(16, 8, 128), (40, 8, 128), (32, 4, 128), (32, 4, 64), (8, 8, 64), (12, 4, 64), (4, 4, 128)])
    case = dict(op=op, nq=nq, nkv=nkv, hd=hd)
    if op != "prefill":
        case["page"] = rng.choice([16, 32, 64, 128])
    if op in ("append", "extend"):
        new = _lengths(rng, _spread(rng, 1, 4000 if op == "append" else 2000), 6)
        past = [rng.choice([0, _spread(rng, 1, 2000)]) for _ in new]
        case.update(bits=16 if op == "append" else 4, new=",".join(map(str, new)), past=",".join(map(str, past)),
                    norm=rng.random() < 0.7)
    elif op == "read":
        case.update(bits=rng.choice([4, 16]), past=",".join(map(str, _lengths(rng, _spread(rng, 16, 40000), 8))))
    elif op == "prefill":
        new = _lengths(rng, _spread(rng, 1, 4000), 6)
        past = [rng.choice([0, 0, _spread(rng, 1, 2000)]) for _ in new]
        case.update(new=",".join(map(str, new)), past=",".join(map(str, past)))
    else:
        case.update(bits=rng.choice([4, 4, 16]),
                    past=",".join(map(str, _lengths(rng, _spread(rng, 16, 60000), rng.choice([1, 4, 32])))))
    return case


def _ints(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------ inputs
def _table(cols, lens, page, gen):
    """A block table over shuffled pages (unused entries name page 0), and the number of pages of the pool."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=gen, device=DEV).int()
    table = torch.zeros(len(lens), max(max(need), cols), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    return table, sum(need) + 3


def _cum(lens):
    return torch.tensor([0] + lens, dtype=torch.int32, device=DEV).cumsum(0).int()


def _keys(gen, t, nkv, hd):
    """Keys as they lie in a cache: unit rows with a few strong channels."""
    strong = 0.5 * torch.randn(nkv, hd, generator=gen, device=DEV)
    return torch.randn(t, nkv, hd, generator=gen, device=DEV) * strong.exp()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, nq, nkv, hd = case["op"], case["nq"], case["nkv"], case["hd"]
    past = _ints(case["past"])
    s = dict(case, past_list=past)

    def f16(*shape):
        return torch.randn(*shape, generator=gen, device=DEV).half()

    if op == "prefill":
        new = _ints(case["new"])
        ctx = [a + b for a, b in zip(past, new)]
        s.update(q=f16(sum(new), nq, hd), k=_keys(gen, sum(ctx), nkv, hd).half(), v=f16(sum(ctx), nkv, hd),
                 cu=_cum(new), cu_k=None if not any(past) else _cum(ctx), most_q=max(new), most_k=max(ctx))
        return s
    page, bits = case["page"], case["bits"]
    new = _ints(case["new"]) if "new" in case else [0] * len(past)
    ctx = [a + b for a, b in zip(past, new)]
    s["table"], pages = _table(1, ctx, page, gen)
    if bits == 16:
        s["k_pages"] = torch.zeros(pages, nkv, page, hd, dtype=torch.float16, device=DEV)
        s["v_pages"] = torch.zeros_like(s["k_pages"])
    else:
        s["k_pages"] = torch.zeros(pages, nkv, page, hd // 2 + hd // 16, dtype=torch.uint8, device=DEV)
        s["v_pages"] = torch.zeros(pages, nkv, page, hd // 2 + 2, dtype=torch.uint8, device=DEV)
    if sum(past):  # what the cache holds already
        b, at = _owner(_cum(past), sum(past))
        _store(s, b, at, _keys(gen, sum(past), nkv, hd).half().float(), f16(sum(past), nkv, hd))
    s["cu_ctx"], s["total"] = _cum(ctx), sum(ctx)
    if op == "decode":
        s.update(q=f16(len(past), nq, hd), lens=torch.tensor(past, dtype=torch.int32, device=DEV), most_k=max(past))
    elif op in ("append", "extend"):
        qkv = f16(sum(new), nq + 2 * nkv, hd)  # one projection's output; the operands are its slices
        s.update(q=qkv[:, :nq], k=qkv[:, nq : nq + nkv], v=qkv[:, nq + nkv :],
                 start=torch.tensor(past, dtype=torch.int32, device=DEV),
                 cu=None if max(new) == 1 else _cum(new), tokens=sum(new))
        angle = (torch.arange(max(ctx) + 5, dtype=torch.float64, device=DEV)[:, None]
                 / 1e6 ** (torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd))
        s.update(cos=angle.cos().float(), sin=angle.sin().float(), eps=1e-6, q_norm=None, k_norm=None)
        if case["norm"]:
            s.update(q_norm=(1 + 0.3 * torch.randn(hd, generator=gen, device=DEV)).half(),
                     k_norm=(0.3 * torch.randn(hd, generator=gen, device=DEV)).exp().half())
    return s


# ------------------------------------------------------------------ plain form: the cache
def _owner(cu, total):
    """Sequence and place within it of each packed row."""
    row = torch.arange(total, device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return b, row - cu[b]


def _parts(s):
    """Views of 4-bit pages: K codes, K scales, V codes (pair, word, which of the pair, two bytes), V scales."""
    kp, vp, page, hd = s["k_pages"], s["v_pages"], s["page"], s["hd"]
    p, h = kp.shape[:2]
    k, v, code = kp.view(p, h, -1), vp.view(p, h, -1), page * hd // 2
    return (k[..., :code].unflatten(-1, (page, hd // 2)), k[..., code:].unflatten(-1, (page, hd // 16)),
            v[..., :code].unflatten(-1, (page // 2, hd // 4, 2, 2)), v[..., code:].unflatten(-1, (page, 2)))


def _quantize(x, group):
    """Codes and fp16 scales of x [..., hd] fp32 in groups."""
    g = x.unflatten(-1, (-1, group))
    scale = (g.abs().amax(-1) / 7).clamp_min(2.0**-14).half()
    code = (g / scale.float()[..., None]).round().clamp(-7, 7).int()
    return code.flatten(-2), scale


def _store(s, b, pos, k, v):
    """Keys k (fp32) and values v (fp16) of rows at positions pos of sequences b into the pages."""
    page, hd = s["page"], s["hd"]
    at, slot = s["table"][b, pos // page].long(), pos % page
    if s["bits"] == 16:
        s["k_pages"][at, :, slot] = k.half()
        s["v_pages"][at, :, slot] = v
        return
    kc, ks, vc, vs = _parts(s)
    code, scale = _quantize(k, GROUP)
    n = code & 15
    n = n.view(*n.shape[:2], hd // 32, 4, 4, 2).transpose(2, 3)  # [rows, heads, t, j, i, odd]
    shift = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=DEV)
    word = (n.long() << shift).sum((-1, -2)).flatten(-2)
    kc[at, :, slot] = torch.stack([word >> 8 * i & 255 for i in range(4)], -1).to(torch.uint8).flatten(-2)
    ks[at, :, slot] = scale.contiguous().view(torch.uint8)
    code, scale = _quantize(v.float(), hd)
    n = (code & 15).unflatten(-1, (hd // 4, 2, 2))  # two bytes of two nibbles
    vc[at, :, slot // 2, :, slot % 2] = (n[..., 0] | n[..., 1] << 4).to(torch.uint8)
    vs[at, :, slot] = scale.contiguous().view(torch.uint8).view(*scale.shape[:2], 2)


def _load(s, b, pos):
    """Keys and values (fp32) at positions pos of sequences b, [rows, heads, hd]."""
    page, hd = s["page"], s["hd"]
    at, slot = s["table"][b, pos // page].long(), pos % page
    if s["bits"] == 16:
        return s["k_pages"][at, :, slot].float(), s["v_pages"][at, :, slot].float()
    kc, ks, vc, vs = _parts(s)
    word = kc[at, :, slot].view(torch.int32).unflatten(-1, (4, hd // 32))[..., None, None]
    shift = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=DEV, dtype=torch.int32)
    k = (((word >> shift) & 15 ^ 8) - 8).transpose(2, 3).flatten(-4).float()
    k = (k.unflatten(-1, (-1, GROUP)) * ks[at, :, slot].view(torch.float16).float()[..., None]).flatten(-2)
    byte = vc[at, :, slot // 2, :, slot % 2].int()
    v = ((torch.stack([byte & 15, byte >> 4], -1) ^ 8) - 8).flatten(-3).float()
    return k, v * vs[at, :, slot].view(torch.float16).float()


def _read(s, b, pos):
    k, v = _load(s, b, pos)
    return k.half(), v.half()


# ------------------------------------------------------------------ plain form: the operators
def _rotate(x, norm, eps, cos, sin):
    """Norm and rotation in fp32; the norm's sum in 64 bits, since a key's code may lie next to a border."""
    x = x.float()
    if norm is not None:
        inv = (1 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()).float()
        x = x * inv * norm.float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    n = s["tokens"]
    if s["cu"] is None:
        b, at = torch.arange(n, device=DEV), torch.zeros(n, dtype=torch.long, device=DEV)
    else:
        b, at = _owner(s["cu"], n)
    pos = s["start"][b] + at
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(s["q"], s["q_norm"], s["eps"], cos, sin)
    k = _rotate(s["k"], s["k_norm"], s["eps"], cos, sin)
    _store(s, b, pos, k, s["v"])
    return q.half(), k.half()


def _prefill(s):
    cu, cu_k = s["cu"].long(), (s["cu"] if s["cu_k"] is None else s["cu_k"]).long()
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    lq, lk = cu.diff(), cu_k.diff()
    iq, ik = torch.arange(s["most_q"], device=DEV), torch.arange(s["most_k"], device=DEV)
    q = s["q"][(cu[:-1, None] + iq).clamp_max(s["q"].shape[0] - 1)].float()
    k = s["k"][(cu_k[:-1, None] + ik).clamp_max(s["k"].shape[0] - 1)].float()
    v = s["v"][(cu_k[:-1, None] + ik).clamp_max(s["v"].shape[0] - 1)].float()
    q = q.transpose(1, 2).unflatten(1, (nkv, nq // nkv)).flatten(2, 3)  # [B, nkv, rep * Lq, hd]
    seen = ik <= iq[:, None] + (lk - lq)[:, None, None]
    x = q @ k.permute(0, 2, 3, 1) / math.sqrt(hd)
    x = x.unflatten(2, (nq // nkv, -1)).masked_fill_(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    o = x.flatten(2, 3) @ v.transpose(1, 2) / x.sum(-1).flatten(2, 3)[..., None]
    o = o.unflatten(2, (nq // nkv, -1)).flatten(1, 2).transpose(1, 2)  # [B, Lq, nq, hd]
    return o[iq < lq[:, None]].half()


def _decode(s):
    nq, nkv, hd, most = s["nq"], s["nkv"], s["hd"], s["most_k"]
    n = s["q"].shape[0]
    pos = torch.arange(most, device=DEV)
    k, v = _load(s, torch.arange(n, device=DEV).repeat_interleave(most), pos.repeat(n))
    k, v = (t.view(n, most, nkv, hd).transpose(1, 2) for t in (k, v))
    x = s["q"].float().view(n, nkv, nq // nkv, hd) @ k.transpose(2, 3) / math.sqrt(hd)
    x = x.masked_fill((pos >= s["lens"][:, None])[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    return (x @ v / x.sum(-1, keepdim=True)).view(n, nq, hd).half()


def run(s):
    op = s["op"]
    if own:
        ops = _ops()
        if op == "prefill":
            return ops.prefill_attention(s["q"], s["k"], s["v"], s["cu"], cu_seqlens_k=s["cu_k"])
        if op == "decode":
            return ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"])
        if op == "read":
            return ops.paged_kv_read(s["k_pages"], s["v_pages"], s["table"], s["cu_ctx"], s["total"])
        q, k = ops.paged_kv_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["cos"],
                                   s["sin"], cu_seqlens=s["cu"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"],
                                   return_k=True)
        if op == "append":
            return q, k, s["k_pages"], s["v_pages"]
        return (q, k, *ops.paged_kv_read(s["k_pages"], s["v_pages"], s["table"], s["cu_ctx"], s["total"]))
    if op == "prefill":
        return _prefill(s)
    if op == "decode":
        return _decode(s)
    if op == "read":
        return _read(s, *_owner(s["cu_ctx"], s["total"]))
    q, k = _append(s)
    if op == "append":
        return q, k, s["k_pages"], s["v_pages"]
    return (q, k, *_read(s, *_owner(s["cu_ctx"], s["total"])))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, nq, nkv, hd = case["op"], case["nq"], case["nkv"], case["hd"]
    past = _ints(case["past"])
    row = 4 * hd if case.get("bits") == 16 else hd + hd // 16 + 2  # a position's key and value of one head
    if op == "decode":
        return {"bytes": sum(past) * nkv * row + 4 * len(past) * nq * hd, "flops": 4 * sum(past) * nq * hd}
    if op == "read":
        return {"bytes": sum(past) * nkv * (row + 4 * hd), "flops": 2 * sum(past) * nkv * hd}
    new = _ints(case["new"])
    t, ctx = sum(new), sum(past) + sum(new)
    if op == "prefill":
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        return {"bytes": 2 * hd * (2 * t * nq + 2 * ctx * nkv), "flops": 4 * pairs * nq * hd}
    tables = 4 * hd * len({p + i for n, p in zip(new, past) for i in range(n)})
    once = 2 * hd * t * (2 * nq + 3 * nkv) + t * nkv * row + tables
    if op == "extend":
        once += ctx * nkv * 4 * hd + sum(past) * nkv * row
    return {"bytes": once, "flops": 10 * t * (nq + nkv) * hd}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rotation(x, norm, eps, cos, sin):
    x = x.double()
    if norm is not None:
        x = x * (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + eps).rsqrt() * norm.double()
    h = x.shape[-1] // 2
    y = torch.empty_like(x)
    y[..., :h] = x[..., :h] * cos - x[..., h:] * sin
    y[..., h:] = x[..., h:] * cos + x[..., :h] * sin
    return y


def _exact_quantized(x, group):
    """What a row in 4 bits stands for; the scale is held in 16 bits by definition."""
    y = torch.empty_like(x)
    for i in range(0, x.shape[-1], group):
        part = x[..., i : i + group]
        scale = torch.clamp_min(part.abs().max(-1, keepdim=True).values / 7, 2.0**-14).half().double()
        y[..., i : i + group] = torch.clamp(torch.round(part / scale), -7, 7) * scale
    return y


def _exact_context(s, b, n):
    """A sequence's first n cached keys and values in 64 bits, [heads, n, hd], nibble by nibble."""
    page, hd, nkv = s["page"], s["hd"], s["nkv"]
    ids = s["table"][b, : -(-n // page)].long()
    if s["bits"] == 16:
        return tuple(t[ids].double().transpose(0, 1).flatten(1, 2)[:, :n] for t in (s["k_pages"], s["v_pages"]))
    k = torch.empty(nkv, len(ids) * page, hd, dtype=torch.float64, device=DEV)
    v = torch.empty_like(k)
    kb, vb = (s[x][ids].transpose(0, 1).flatten(2) for x in ("k_pages", "v_pages"))  # [heads, pages, bytes]
    code = page * hd // 2
    ksc = kb[..., code:].contiguous().view(torch.float16).double().reshape(nkv, -1, hd // GROUP)
    vsc = vb[..., code:].contiguous().view(torch.float16).double().reshape(nkv, -1)
    kcode = kb[..., :code].reshape(nkv, -1, hd // 2)
    vcode = vb[..., :code].reshape(nkv, -1, hd)  # a row of bytes for two positions
    for d in range(hd):
        j, t, e = d // 32, d % 32 // 8, d % 8
        nibble = e // 2 + 4 * (e % 2)
        x = kcode[..., 4 * (t * (hd // 32) + j) + nibble // 2] >> 4 * (nibble % 2) & 15
        k[..., d] = torch.where(x > 7, x.double() - 16, x.double()) * ksc[..., d // GROUP]
        for odd in range(2):
            x = vcode[..., d // 4 * 4 + 2 * odd + d % 4 // 2] >> 4 * (d % 2) & 15
            v[:, odd::2, d] = torch.where(x > 7, x.double() - 16, x.double()) * vsc[:, odd::2]
    return k[:, :n], v[:, :n]


def _exact_attention(q, k, v, first):
    """q [rows, heads, hd] over k, v [kv heads, n, hd]; row i sees keys up to first + i."""
    rep, out = q.shape[1] // k.shape[0], torch.empty(q.shape, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // k.shape[1])
    for h in range(q.shape[1]):
        for i in range(0, q.shape[0], step):
            x = q[i : i + step, h].double() @ k[h // rep].t() / math.sqrt(q.shape[2])
            rows = torch.arange(i, i + x.shape[0], device=DEV)
            hidden = torch.arange(k.shape[1], device=DEV) > first + rows[:, None]
            out[i : i + step, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // rep]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, past = s["op"], s["past_list"]
    if op == "decode":
        return torch.cat([_exact_attention(s["q"][b : b + 1], *_exact_context(s, b, n), n - 1) for b, n in enumerate(past)])
    if op == "read":
        ctx = [_exact_context(s, b, n) for b, n in enumerate(past)]
        return tuple(torch.cat([c[i] for c in ctx], 1).transpose(0, 1).contiguous() for i in range(2))
    new = _ints(case["new"])
    if op == "prefill":
        out, iq, ik = [], 0, 0
        for n, p in zip(new, past):
            k, v = (s[x][ik : ik + n + p].double().transpose(0, 1) for x in ("k", "v"))
            out.append(_exact_attention(s["q"][iq : iq + n], k, v, p))
            iq, ik = iq + n, ik + n + p
        return torch.cat(out)
    qs, ks, held, at = [], [], [], 0
    if op == "append":
        held = [s["k_pages"].double(), s["v_pages"].double()]
    for b, (n, p) in enumerate(zip(new, past)):
        rows = slice(at, at + n)
        cos, sin = (s[x][p : p + n, None].double() for x in ("cos", "sin"))
        q = _exact_rotation(s["q"][rows], s["q_norm"], s["eps"], cos, sin)
        k = _exact_rotation(s["k"][rows], s["k_norm"], s["eps"], cos, sin)
        v = s["v"][rows].double()
        qs.append(q)
        ks.append(k)
        if op == "append":
            place = torch.arange(p, p + n, device=DEV)
            ids, slot = s["table"][b].long()[place // s["page"]], place % s["page"]
            held[0][ids, :, slot] = k
            held[1][ids, :, slot] = v
        else:
            ck, cv = _exact_context(s, b, p)
            held.append((torch.cat([ck, _exact_quantized(k, GROUP).transpose(0, 1)], 1),
                         torch.cat([cv, _exact_quantized(v, s["hd"]).transpose(0, 1)], 1)))
        at += n
    if op == "append":
        return torch.cat(qs), torch.cat(ks), *held
    return (torch.cat(qs), torch.cat(ks),
            *(torch.cat([h[i] for h in held], 1).transpose(0, 1).contiguous() for i in range(2)))
