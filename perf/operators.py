"""Serving from a paged key/value cache held in 4 bits: what is measured, and each operator's plain form.

Four operators that a serving loop runs in turn:

* plan    block table, slot map and positions for the next step's tokens, from the requests' lengths;
* append  new keys and values quantised into the cache (the pass reads them back, as values);
* read    cached keys and values as dense 16-bit tensors;
* attend  attention of new queries over the cache.

The cache holds groups of 64 values of one token's head vector as `s * (c - z)`: codes c and a zero
point z in 0..15, a scale s of 4 significant bits. Sixteen tokens form a block of 32-bit words (128
words of codes for each group, then 8 words of 16-bit `scale | zero point` for each group); pages are
`[page, keys or values, head, block]`.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
FLOOR = {"bf16": 2.0 ** -126, "fp16": 2.0 ** -21}  # smallest scale


# ------------------------------------------------------------------ cases

def listed():
    return [
        # One decode step of a small batch: every request gets one token, few need a page. Latency alone.
        dict(name="plan_decode_b8", op="plan", b=8, n=1, pages=64, page=64, lo=1, hi=4000, share=0.0),
        # A busy server's step: decodes, prompts' chunks of up to 512 tokens and finished requests together.
        dict(name="plan_mixed_b256", op="plan", b=256, n=512, pages=512, page=64, lo=0, hi=32000, share=0.3),
        # One token of 64 requests into a global layer's cache (head_dim 512, 4 KV heads).
        dict(name="append_decode_b64", op="append", b=64, hkv=4, d=512, n=1, page=64, dtype="bf16", lo=1, hi=1),
        # A long prompt of two requests into a sliding layer's cache (head_dim 256, 8 KV heads).
        dict(name="append_prompt_d256", op="append", b=2, hkv=8, d=256, n=8192, page=64, dtype="bf16", lo=8192, hi=8192),
        # Ragged chunks, an odd batch, short pages, fp16.
        dict(name="append_ragged_d128", op="append", b=7, hkv=4, d=128, n=1021, page=16, dtype="fp16", lo=0, hi=1021),
        # A cached prefix of one request, shared by a new prompt.
        dict(name="read_prefix_d512", op="read", b=1, hkv=4, d=512, n=4096, page=64, dtype="bf16", lo=4001, hi=4096),
        # Caches of an odd batch back to 16 bits, short pages, fp16.
        dict(name="read_ragged_d128", op="read", b=5, hkv=8, d=128, n=16384, page=16, dtype="fp16", lo=100, hi=16384),
        # One token of one request on a sliding layer: the smallest attention, latency alone.
        dict(name="attend_swa_b1", op="attend", b=1, hq=16, hkv=8, d=256, n=1, page=64, dtype="bf16", window=512,
             lo=900, hi=1000, cap=1024),
        # One token of 16 requests on a global layer with up to 16K cached tokens.
        dict(name="attend_global_b16", op="attend", b=16, hq=32, hkv=4, d=512, n=1, page=64, dtype="bf16", window=0,
             lo=8192, hi=16384, cap=16384),
        # One token of one request with a long cache.
        dict(name="attend_long_b1", op="attend", b=1, hq=16, hkv=2, d=512, n=1, page=128, dtype="bf16", window=0,
             lo=130000, hi=131072, cap=131072),
        # Five drafted tokens to verify, odd batch, short pages, fp16.
        dict(name="attend_verify_d128", op="attend", b=7, hq=32, hkv=8, d=128, n=5, page=16, dtype="fp16", window=0,
             lo=5, hi=8191, cap=8192),
        # A prompt's chunk of 1024 tokens behind cached ones on a global layer.
        dict(name="attend_chunk_d512", op="attend", b=2, hq=32, hkv=4, d=512, n=1024, page=64, dtype="bf16", window=0,
             lo=6000, hi=8192, cap=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "read", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        n = _log(rng, 1, 512)
        pages = max(2, _log(rng, 512, 32768) // page)
        b = _log(rng, 1, 256)
        return dict(op=op, b=b, n=n, pages=pages, page=page, lo=0, hi=max(1, int(pages * page * rng.uniform(0.3, 1.0))),
                    share=rng.choice([0.0, 0.2, 0.5]))
    d = rng.choice([64, 128, 256, 512])
    dtype = rng.choice(["bf16", "fp16"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    if op in ("append", "read"):
        n = _log(rng, 1, 16384)
        b = max(1, min(_log(rng, 1, 128), 2 * 8 * 256 * 8192 // (n * hkv * d)))
        return dict(op=op, b=b, hkv=hkv, d=d, n=n, page=page, dtype=dtype, lo=rng.choice([0, n // 2, n]), hi=n)
    g = rng.choice([1, 2, 3, 4, 7, 8])
    n = rng.choice([1, 1, 2, 3, 5, 8, _log(rng, 9, 1024)])
    cap = max(n, _log(rng, 16, 131072))
    most = min(16 * 16384 * 4 * 512 // (cap * hkv * d), 2 * 32 * 1024 * 8192 // (cap * n * g * hkv))
    while most < 1:
        cap //= 2
        n = min(n, cap)
        most = min(16 * 16384 * 4 * 512 // (cap * hkv * d), 2 * 32 * 1024 * 8192 // (cap * n * g * hkv))
    b = max(1, min(_log(rng, 1, 64), most))
    window = rng.choice([0, 0, _log(rng, 1, max(2, cap))])
    return dict(op=op, b=b, hq=g * hkv, hkv=hkv, d=d, n=n, page=page, dtype=dtype, window=window,
                lo=rng.choice([0, cap // 2, cap]), hi=cap, cap=cap)


# ------------------------------------------------------------------ inputs

def _lengths(b, lo, hi, rng):
    """b lengths spread evenly over [lo, hi], in an order that the seed gives."""
    at = lo + (hi - lo) * (np.arange(b) + rng.uniform(0.3, 0.7, b)) / b
    return torch.from_numpy(rng.permutation(np.rint(at).astype(np.int32)))


def _normal(shape, gen, dt):
    """Unit normal values, with a few channels of several times the others' size, as keys have them."""
    d = shape[-1]
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    size = 1.0 + 3.0 * (torch.rand(d, generator=gen, device="cuda") > 0.97).float()
    return (x * size).to(dt)


def _logical(case, seed):
    """Inputs by what they mean, before they are laid out: lengths on the host, values on the GPU."""
    rng = np.random.RandomState(seed % (2 ** 32))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, b, page = case, case["b"], case["page"]
    if c["op"] == "plan":
        lens = _lengths(b, c["lo"], min(c["hi"], c["pages"] * page), rng).numpy()
        kind = rng.uniform(size=b)
        new = np.ones(b, np.int32)
        new[kind < c["share"]] = rng.randint(0, c["n"] + 1, int((kind < c["share"]).sum()))
        new[kind < c["share"] / 5] = -1  # finished
        used = -(-lens // page)
        total = b * -(-min(c["hi"], c["pages"] * page) // page) + 2 * b + b * c["n"] // page // 2 + 8
        # free pages: at times too few for every request (other requests hold the rest)
        count = int((2 * b + b * c["n"] // page // 2) * (rng.uniform(0.05, 1.0) if c["share"] else 1.0)) + 8
        perm = rng.permutation(total).astype(np.int32)
        table = np.full((b, c["pages"]), -1, np.int32)
        at = np.concatenate([[0], np.cumsum(used)])
        for i in range(b):
            table[i, :used[i]] = perm[at[i]:at[i + 1]]
        free = np.full(total, -1, np.int32)
        head = int(rng.randint(total))
        free[(head + np.arange(count)) % total] = perm[at[-1]:at[-1] + count]
        return dict(lens=lens, new=new, table=table, free=free, state=np.array([head, count], np.int32))
    dt = DT[c["dtype"]]
    if c["op"] == "append":
        new = _lengths(b, c["lo"], c["hi"], rng)
        start = torch.from_numpy(rng.randint(0, 200, b).astype(np.int32))
        k, v = (_normal((b, c["n"], c["hkv"], c["d"]), gen, dt).transpose(1, 2) for _ in range(2))
        return dict(start=start, lens=start + new, new=new, k=k, v=v, cap=200 + c["n"], rng=rng)
    cap = c["n"] if c["op"] == "read" else c["cap"]
    lens = _lengths(b, c["lo"], c["hi"], rng)
    k, v = (_quantise(_normal((b, c["hkv"], cap, c["d"]), gen, dt), c["dtype"]) for _ in range(2))
    got = dict(lens=lens, k=k, v=v, cap=cap, rng=rng)
    if c["op"] == "attend":
        got["q"] = _normal((b, c["n"], c["hq"], c["d"]), gen, dt).transpose(1, 2)
        got["new"] = torch.minimum(torch.from_numpy(rng.randint((c["n"] + 1) // 2, c["n"] + 1, b).astype(np.int32)), lens)
    return got


def prepare(case, seed):
    c = case
    x = _logical(c, seed)
    if c["op"] == "plan":
        s = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in x.items()}
        s["case"] = c
        return s
    rng = x.pop("rng")
    cols = max(1, -(-x["cap"] // c["page"]))
    total = c["b"] * cols + 3
    table = torch.from_numpy(rng.permutation(total)[:c["b"] * cols].astype(np.int32).reshape(c["b"], cols)).cuda()
    words = c["d"] // 64 * 136
    pages = torch.zeros((total, 2, c["hkv"], c["page"] // 16, words), dtype=torch.int32, device="cuda")
    s = dict(case=c, table=table, pages=pages, lens=x["lens"].cuda(), start=torch.zeros_like(x["lens"]).cuda())
    if c["op"] == "append":
        s.update(start=x["start"].cuda(), k=x["k"], v=x["v"])
        pos = torch.arange(c["n"], device="cuda")[None, :] + s["start"][:, None]
        slots = torch.gather(table, 1, (pos // c["page"]).long()) * c["page"] + pos % c["page"]
        s["slots"] = torch.where(pos < s["lens"][:, None], slots, torch.full_like(slots, -1)).int()
    else:
        pos = torch.arange(x["cap"], device="cuda")[None, :].expand(c["b"], -1)
        slots = torch.gather(table, 1, pos // c["page"]).long() * c["page"] + pos % c["page"]
        for kind, key in enumerate("kv"):
            codes, scale, zero = x.pop(key)
            _store(pages, c, kind, slots, codes.transpose(1, 2), scale.transpose(1, 2), zero.transpose(1, 2))
        if c["op"] == "attend":
            s.update(q=x["q"], new=x["new"].cuda())
    s["cache"] = _cache(pages, c) if own else None
    return s


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma-triton-flash-attn_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gemma_triton_flash_attn

    return gemma_triton_flash_attn


def _cache(pages, c):
    return _package().KV4Cache(pages.view(torch.uint8), head_dim=c["d"], page_size=c["page"], dtype=DT[c["dtype"]])


# ------------------------------------------------------------------ the plain forms

def _quantise(x, dtype):
    """Codes [..., d], scales and zero points [..., d / 64] of 16-bit values, in 32 bits. A group with a value
    that is not finite gets a scale that is not a number."""
    x = x.float().unflatten(-1, (-1, 64))
    top, low = x.amax(-1, keepdim=True).clamp_min(0), x.amin(-1, keepdim=True).clamp_max(0)
    step = (top * 0.5 - low * 0.5) / torch.full_like(top, 7.5)  # a quotient, not a product with 1 / 7.5
    up = ((step.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32)  # up to 4 significant bits
    scale = up.clamp_min(FLOOR[dtype])
    zero = torch.floor(-low / scale + 0.5)
    code = (torch.floor(x / scale + 0.5) + zero).clamp_max(15)
    far = scale * (code - zero)
    most = torch.finfo(DT[dtype]).max
    code = code - (far > most).float() + (far < -most).float()
    fine = torch.isfinite(x).all(-1, keepdim=True)
    code, zero = torch.where(fine, code, torch.zeros_like(code)), torch.where(fine, zero, torch.zeros_like(zero))
    scale = torch.where(fine, scale, torch.full_like(scale, math.nan))
    return code.to(torch.uint8).flatten(-2), scale.squeeze(-1), zero.squeeze(-1).to(torch.uint8)


def _places(c, kind, slots):
    """Indices of 32-bit code words [..., heads, groups, 8] and of 16-bit meta words [..., heads, groups]."""
    dev = slots.device
    groups, page = c["d"] // 64, c["page"]
    s = slots[..., None, None]
    head = torch.arange(c["hkv"], device=dev)[:, None]
    base = (((s // page * 2 + kind) * c["hkv"] + head) * (page // 16) + s % page // 16) * (groups * 136)
    r = s % 16
    grp = torch.arange(groups, device=dev)
    j = torch.arange(8, device=dev)
    r8, grp8 = r[..., None], grp[:, None]
    if kind == 0:
        word = r8 % 8 * 16 + j // 2 * 4 + r8 // 8 * 2 + j % 2
        meta = r % 8 * 2 + r // 8
    else:
        t = r8 % 8 // 2
        word = (t * 8 + (j ^ (2 * t))) * 4 + r8 // 8 * 2 + r8 % 2
        meta = r % 8 // 2 * 4 + r // 8 * 2 + r % 2
    return base[..., None] + grp8 * 128 + word, base * 2 + groups * 256 + grp * 16 + meta


#: Place of a word's eight values in its nibbles, lowest first: keys pair neighbours over the halves.
NIBBLE = {0: [0, 2, 4, 6, 1, 3, 5, 7], 1: [0, 1, 2, 3, 4, 5, 6, 7]}


def _store(pages, c, kind, slots, codes, scale, zero):
    """Lays codes [..., heads, d], scales and zero points [..., heads, groups] out at `slots` [...]."""
    word, meta = _places(c, kind, slots.long())
    shift = torch.arange(0, 32, 4, device=codes.device)
    x = codes.unflatten(-1, (-1, 8, 8))[..., NIBBLE[kind]]
    packed = (x.long() << shift).sum(-1)
    packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()
    bits = (scale.contiguous().view(torch.int32) >> 16 & 0xFFF0 | zero.int())
    bits = torch.where(torch.isnan(scale), torch.full_like(bits, 0x7FF0), bits)
    pages.view(-1)[word.reshape(-1)] = packed.reshape(-1)
    pages.view(-1).view(torch.int16)[meta.reshape(-1)] = bits.to(torch.int16).reshape(-1)


def _load(pages, c, kind, slots):
    """Values [..., heads, d] in 32 bits of the tokens at `slots` [...]."""
    word, meta = _places(c, kind, slots.long())
    shift = torch.arange(0, 32, 4, device=slots.device, dtype=torch.int32)
    code = (pages.view(-1)[word][..., None] >> shift & 15).to(torch.uint8)
    back = torch.argsort(torch.tensor(NIBBLE[kind], device=slots.device))
    bits = pages.view(-1).view(torch.int16)[meta].int()
    scale = ((bits & 0xFFF0) << 16).view(torch.float32)
    zero = (bits & 15).float()
    return ((code[..., back].flatten(-2).float() - zero[..., None]) * scale[..., None]).flatten(-2)


def _gather(s, start, n):
    """Keys and values [b, heads, n, d] in 32 bits of positions start .. start + n, zeros behind a request's last."""
    c = s["case"]
    pos = start[:, None] + torch.arange(n, device=start.device)[None, :]
    live = pos < s["lens"][:, None]
    at = torch.where(live, pos, torch.zeros_like(pos)).long()
    slots = torch.gather(s["table"], 1, at // c["page"]).long() * c["page"] + at % c["page"]
    keep = live[:, :, None, None]
    return [torch.where(keep, _load(s["pages"], c, kind, slots), torch.zeros((), device=pos.device)).transpose(1, 2)
            for kind in (0, 1)]


def _plan(s):
    c, lens, new, table, free = s["case"], s["lens"], s["new"], s["table"], s["free"]
    page, total = c["page"], free.numel()
    head, count = s["state"][0], s["state"][1]
    gone = new < 0
    ok = (new <= c["n"]) & (lens + new <= c["pages"] * page)
    used = (lens + page - 1) // page
    need = torch.where(ok & ~gone, (lens + new.clamp_min(0) + page - 1) // page - used, torch.zeros_like(lens))
    upto = torch.cumsum(need, 0).int()
    ok = ok & ((need == 0) | (upto <= count))
    need = torch.where(ok, need, torch.zeros_like(need))
    given = torch.where(ok & ~gone, new, torch.zeros_like(new))
    out_lens = torch.where(gone, torch.zeros_like(lens), lens + given)
    col = torch.arange(c["pages"], device=lens.device)[None, :]
    fresh = col - used[:, None]
    is_new = (fresh >= 0) & (fresh < need[:, None])
    at = (head + (upto - need)[:, None] + fresh) % total
    rows = torch.where(col < used[:, None], table, torch.full_like(table, -1))
    rows = torch.where(is_new, free[at.long()], rows)
    rows = torch.where(gone[:, None], torch.full_like(rows, -1), rows)
    i = torch.arange(c["n"], device=lens.device)[None, :]
    live = i < given[:, None]
    pos = torch.where(live, lens[:, None] + i, torch.full_like(live, -1, dtype=torch.int32)).int()
    slot = torch.gather(rows, 1, (pos.clamp_min(0) // page).long()) * page + pos % page
    slot = torch.where(live, slot, torch.full_like(slot, -1))
    back = torch.where(gone, used, torch.zeros_like(used))
    taken = need.sum().int()
    state = torch.stack([(head + taken) % total, count - taken + back.sum().int()])
    ring = free.clone()
    where = head + count + (torch.cumsum(back, 0).int() - back)[:, None] + col
    mine = gone[:, None] & (col < used[:, None])
    ring[(where % total)[mine].long()] = table[mine]
    return dict(block_table=rows, kv_lens=out_lens, new_lens=given, slot_map=slot, positions=pos, free_pages=ring,
                free_state=state, accepted=ok.int())


def _attend(s):
    c, q, lens, new = s["case"], s["q"], s["lens"], s["new"]
    k, v = _gather(s, s["start"], c["cap"])
    b, g = c["b"], c["hq"] // c["hkv"]
    qq = q.float().reshape(b, c["hkv"], g, c["n"], c["d"])
    score = torch.matmul(qq.flatten(2, 3), k.transpose(-1, -2)) * c["d"] ** -0.5
    score = score.unflatten(2, (g, c["n"]))
    i = torch.arange(c["n"], device=q.device)[None, :, None]
    at = (lens - new)[:, None, None] + i
    key = torch.arange(c["cap"], device=q.device)[None, None, :]
    seen = (key <= at) & (i < new[:, None, None])
    if c["window"]:
        seen = seen & (key > at - c["window"])
    seen = seen[:, None, None]
    score = torch.where(seen, score, torch.full((), -math.inf, device=q.device))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (g, c["n"]))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.flatten(1, 2).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        gfa = _package()
        if c["op"] == "plan":
            p = gfa.kv4_plan(s["lens"], s["new"], s["table"], s["free"], s["state"], page_size=c["page"],
                             max_new=c["n"])
            return dict(block_table=p.block_table, kv_lens=p.kv_lens, new_lens=p.new_lens, slot_map=p.slot_map,
                        positions=p.positions, free_pages=s["free"], free_state=p.free_state, accepted=p.accepted)
        if c["op"] == "append":
            gfa.kv4_append(s["cache"], s["k"], s["v"], s["slots"])
        if c["op"] in ("append", "read"):
            return list(gfa.kv4_read(s["cache"], s["table"], s["lens"], c["n"], starts=s["start"]))
        return gfa.attention_flash_gqa_kv4(s["q"], s["cache"], s["table"], s["lens"], causal=True,
                                           slide_size=c["window"], q_lens=s["new"], max_kv_len=c["cap"])
    if c["op"] == "plan":
        return _plan(s)
    if c["op"] == "append":
        keep = s["slots"] >= 0
        for kind, key in enumerate("kv"):
            x = s[key].transpose(1, 2)[keep]
            _store(s["pages"], c, kind, s["slots"][keep], *_quantise(x, c["dtype"]))
    if c["op"] in ("append", "read"):
        return [x.to(DT[c["dtype"]]) for x in _gather(s, s["start"], c["n"])]
    return _attend(s)


# ------------------------------------------------------------------ work, and 64-bit results

def work(case):
    c = case
    if c["op"] == "plan":
        # table in and out, slots and positions out; lengths, ring and flags are small beside them
        return {"bytes": 4 * (2 * c["b"] * c["pages"] + 2 * c["b"] * c["n"] + 6 * c["b"]), "flops": 0}
    mean = (c["lo"] + c["hi"]) / 2
    full = 2 * c["hkv"] * c["d"] * 2  # bytes of a token's keys and values in 16 bits
    held = full * 17 / 64
    if c["op"] == "append":
        return {"bytes": c["b"] * (mean * (full + 2 * held) + c["n"] * full), "flops": 0}
    if c["op"] == "read":
        return {"bytes": c["b"] * (mean * held + c["n"] * full), "flops": 0}
    new = min(mean, (3 * c["n"] + 1) / 4)
    seen = max(1.0, mean - (new - 1) / 2)
    span = mean
    if c["window"]:
        seen, span = min(seen, c["window"]), min(span, c["window"] + new - 1)
    qo = 2 * c["b"] * c["hq"] * c["n"] * c["d"] * 2
    return {"bytes": c["b"] * span * held + qo, "flops": 4 * c["b"] * new * seen * c["hq"] * c["d"]}


def _exact_plan(c, x):
    lens, new, table, free = (x[k].astype(np.int64) for k in ("lens", "new", "table", "free"))
    head, count = (int(v) for v in x["state"])
    b, page, total = c["b"], c["page"], free.size
    out = dict(block_table=np.full((b, c["pages"]), -1, np.int32), kv_lens=np.zeros(b, np.int32),
               new_lens=np.zeros(b, np.int32), slot_map=np.full((b, c["n"]), -1, np.int32),
               positions=np.full((b, c["n"]), -1, np.int32), accepted=np.zeros(b, np.int32))
    ring, asked, taken, back = free.astype(np.int32).copy(), 0, 0, 0
    for i in range(b):
        used = -(-int(lens[i]) // page)
        if new[i] < 0:
            for j in range(used):
                ring[(head + count + back) % total] = table[i, j]
                back += 1
            out["accepted"][i] = 1
            continue
        out["block_table"][i, :used] = table[i, :used]
        out["kv_lens"][i] = lens[i]
        if new[i] > c["n"] or lens[i] + new[i] > c["pages"] * page:
            continue
        need = -(-int(lens[i] + new[i]) // page) - used
        asked += need
        if need and asked > count:
            continue
        for j in range(need):
            out["block_table"][i, used + j] = free[(head + taken) % total]
            taken += 1
        out["accepted"][i], out["new_lens"][i] = 1, new[i]
        out["kv_lens"][i] += new[i]
        for j in range(int(new[i])):
            p = int(lens[i]) + j
            out["positions"][i, j] = p
            out["slot_map"][i, j] = out["block_table"][i, p // page] * page + p % page
    out["free_pages"] = ring
    out["free_state"] = np.array([(head + taken) % total, count - taken + back], np.int32)
    return {k: torch.from_numpy(v) for k, v in out.items()}


def _round_trip(x, dtype):
    """What 16-bit values become in the cache, from the definition in 64 bits."""
    x = x.double().unflatten(-1, (-1, 64))
    top, low = x.amax(-1, keepdim=True).clamp(min=0), x.amin(-1, keepdim=True).clamp(max=0)
    m, e = torch.frexp((top - low) / 15)
    scale = torch.ldexp(torch.ceil(m * 16) / 16, e).clamp(min=FLOOR[dtype])
    zero = torch.floor(0.5 - low / scale)
    code = torch.minimum(torch.floor(x / scale + 0.5) + zero, torch.full_like(x, 15))
    return ((code - zero) * scale).flatten(-2)


def exact(case, seed):
    c = case
    x = _logical(c, seed)
    if c["op"] == "plan":
        return _exact_plan(c, x)
    lens = x["lens"].cuda()
    if c["op"] == "append":
        live = torch.arange(c["n"], device="cuda")[None, :] < x["new"].cuda()[:, None]
        return [torch.where(live[:, None, :, None], _round_trip(x[k], c["dtype"]), 0.0) for k in "kv"]

    def values(key, i, h):
        code, scale, zero = (t[i, h] for t in x[key])
        per = code.double().reshape(code.shape[0], -1, 64) - zero.double()[..., None]
        return (per * scale.double()[..., None]).reshape(code.shape)

    b, hkv, n, d = c["b"], c["hkv"], c["n"], c["d"]
    if c["op"] == "read":
        out = [torch.zeros((b, hkv, n, d), dtype=torch.float64, device="cuda") for _ in range(2)]
        for i in range(b):
            for h in range(hkv):
                for o, key in zip(out, "kv"):
                    o[i, h, :lens[i]] = values(key, i, h)[:lens[i]]
        return out
    g = c["hq"] // hkv
    out = torch.zeros((b, c["hq"], n, d), dtype=torch.float64, device="cuda")
    for i in range(b):
        length, new = int(x["lens"][i]), int(x["new"][i])
        if new == 0:
            continue
        at = length - new + torch.arange(new, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        hide = key > at
        if c["window"]:
            hide |= key <= at - c["window"]
        for h in range(hkv):
            k, v = values("k", i, h)[:length], values("v", i, h)[:length]
            for j in range(g):
                w = (x["q"][i, h * g + j, :new].double() @ k.T) / math.sqrt(d)
                out[i, h * g + j, :new] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v
    return out
