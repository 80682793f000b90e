"""A second question on a cached picture, and a cache that gives up what nobody looks at, as measurable cases.

A case is a dict of plain values; ``op`` names the public entry point that one pass goes through:

* ``chunk``   ``ops.chunk_attention``: several new tokens at once over [system | 4-bit visual | text], with the log-sum-exp;
* ``weights`` ``ops.key_weights``: how much attention those queries paid to every cached key, per KV head;
* ``groups``  ``ops.evict_groups``: the groups of 32 visual tokens with the largest weight stay, packed as they are;
* ``tokens``  ``ops.evict_tokens``: the same for single full-precision tokens, system and recent ones always staying.

Token counts: 41 system tokens, 256 visual tokens per image tile (13 tiles = 3328), head dim 128, 8 KV heads with 4 or 6 query
heads each.  Keys carry outlier channels (per-channel lognormal factor); the visual span is quantized here as the packs do it:
keys per channel, values per token, groups of 32.
"""

from __future__ import annotations

import math

import torch

own = False

D, HKV, SYS, GROUP, LEVELS = 128, 8, 41, 32, 15
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a thumbnail and a few words: one token of one request, where latency counts
        dict(name="chunk_b1_n1_t256", op="chunk", batch=1, new=1, vis=256, text=23, rep=4, dtype="fp16", mask=False),
        # the 7B backbone's serving step when the weights of the keys are tracked: one token of each of 16 requests, 13 tiles
        dict(name="chunk_b16_n1_t3328", op="chunk", batch=16, new=1, vis=3328, text=151, rep=4, dtype="bf16", mask=False),
        # a second question of a sentence to two large pictures of the 20B backbone, padded requests (additive mask)
        dict(name="chunk_b4_n37_t6656_masked", op="chunk", batch=4, new=37, vis=6656, text=190, rep=6, dtype="bf16", mask=True),
        # a paragraph after five tiles and a little more, odd sizes
        dict(name="chunk_b2_n517_t1312", op="chunk", batch=2, new=517, vis=1312, text=83, rep=4, dtype="fp16", mask=False),
        # a document pasted into eight running chats
        dict(name="chunk_b8_n1024_t3328", op="chunk", batch=8, new=1024, vis=3328, text=215, rep=4, dtype="bf16", mask=False),
        # tracking behind the smallest step
        dict(name="weights_b1_n1_t256", op="weights", batch=1, new=1, vis=256, text=23, rep=4, dtype="fp16", mask=False),
        # tracking behind the serving step
        dict(name="weights_b16_n1_t3328", op="weights", batch=16, new=1, vis=3328, text=151, rep=4, dtype="bf16", mask=False),
        # tracking behind the pasted document
        dict(name="weights_b8_n1024_t3328", op="weights", batch=8, new=1024, vis=3328, text=215, rep=4, dtype="bf16", mask=False),
        # five tiles of one request, half of the groups go
        dict(name="groups_b1_t1280", op="groups", batch=1, vis=1280, keep=20, dtype="bf16"),
        # long contexts of eight requests, a quarter of the groups stays
        dict(name="groups_b8_t32768", op="groups", batch=8, vis=32768, keep=256, dtype="fp16"),
        # the text of one chat
        dict(name="tokens_b1_t301", op="tokens", batch=1, text=301, keep=160, recent=32, dtype="bf16"),
        # long chats of 16 requests
        dict(name="tokens_b16_t4099", op="tokens", batch=16, text=4099, keep=1024, recent=256, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "weights", "weights", "groups", "tokens"])
    dtype = rng.choice(["fp16", "bf16"])
    biggest = {c["op"]: work(c) for c in listed()}      # the last listed case of an operator is its largest
    while True:
        batch = _log(rng, 1, 16)
        if op in ("chunk", "weights"):
            new = _log(rng, 1, 1100)
            text = SYS + new + _log(rng, 1, 600)
            case = dict(op=op, batch=batch, new=new, vis=GROUP * _log(rng, 1, 400), text=text, rep=rng.choice([1, 2, 4, 6, 8]),
                        dtype=dtype, mask=rng.random() < 0.3)
            case["text"] -= SYS + new                     # what is neither system prompt nor new
        elif op == "groups":
            groups = _log(rng, 2, 1100)
            case = dict(op=op, batch=batch, vis=GROUP * groups, keep=_log(rng, 1, groups), dtype=dtype)
        else:
            text = _log(rng, 64, 5000)
            recent = rng.randint(0, (text - SYS) // 2)
            case = dict(op=op, batch=batch, text=text, recent=recent, keep=rng.randint(SYS + recent, text), dtype=dtype)
        w = work(case)
        if all(w[k] <= biggest[op][k] for k in w):
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _pack(x):
    """4-bit groups of 32 along the last dimension: (code int32 [.., L/8], scale [.., L/32], mn [.., L/32])."""
    g = x.unflatten(-1, (-1, GROUP))
    mn = g.amin(-1)
    scale = (g.amax(-1) - mn) / LEVELS
    code = ((g - mn.unsqueeze(-1)) / scale.clamp_min(1e-6).unsqueeze(-1)).clamp(0, LEVELS).round().to(torch.int32).unflatten(-1, (-1, 8))
    word = code[..., 0].clone()
    for i in range(1, 8):
        word |= code[..., i] << (4 * i)
    return word.flatten(-2), scale, mn


def _cache(case, gen, dev):
    """Packed visual span and full-precision tokens, built a request at a time (the unpacked span of all would be large)."""
    dt, B = DT[case["dtype"]], case["batch"]
    t_fp = SYS + case["text"] + case["new"] if "new" in case else case.get("text", 0)
    channel = torch.exp(torch.randn(D, generator=gen, device=dev))
    parts = [[], []]
    for _ in range(B if case.get("vis") else 0):
        k = (torch.randn(1, HKV, case["vis"], D, generator=gen, device=dev) * channel).to(dt)
        v = torch.randn(1, HKV, case["vis"], D, generator=gen, device=dev).to(dt)
        parts[0].append(_pack(k.transpose(2, 3).contiguous()))
        parts[1].append(_pack(v))
    packs = [tuple(torch.cat(t) for t in zip(*p)) for p in parts] if parts[0] else [None, None]
    k_fp = (torch.randn(B, HKV, t_fp, D, generator=gen, device=dev) * channel).to(dt)
    v_fp = torch.randn(B, HKV, t_fp, D, generator=gen, device=dev).to(dt)
    return packs[0], packs[1], k_fp, v_fp


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, B = DT[case["dtype"]], case["batch"]
    s = {"case": case}
    s["k_pack"], s["v_pack"], s["k_fp"], s["v_fp"] = _cache(case, gen, dev)
    if case["op"] in ("chunk", "weights"):
        s["q"] = torch.randn(B, case["new"], HKV * case["rep"], D, generator=gen, device=dev).to(dt)
        s["mask"] = None
        if case["mask"]:      # requests of other lengths, padded: a run of tokens in front of the new ones does not count
            n = SYS + case["vis"] + case["text"] + case["new"]
            m = torch.zeros(B, n, device=dev)
            for b in range(B):
                pad = int(torch.randint(0, case["text"] + 1, (1,), generator=gen, device=dev))
                end = n - case["new"]
                m[b, end - pad:end] = -math.inf if b % 2 else torch.finfo(dt).min
            s["mask"] = m.to(dt)
        if case["op"] == "weights":
            s["lse"] = _plain_chunk(s)[1]      # what the attention call before it gave
    else:
        n = case["vis"] if case["op"] == "groups" else case["text"]
        w = torch.exp(2.7 * torch.randn(B, HKV, n, generator=gen, device=dev)) * 1e-3
        s["weights"] = w * (torch.rand(B, HKV, n, generator=gen, device=dev) > 0.1)      # some were never looked at: ties
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _unpack(pack):
    """float32 values of a packed operand."""
    code, scale, mn = pack
    c = torch.stack([(code >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (c * scale.float().unsqueeze(-1) + mn.float().unsqueeze(-1)).flatten(-2)


def _requests(s):
    """Slices of the batch whose scores, all heads of them, take half a gigabyte at most (one request at least)."""
    case = s["case"]
    step = max(1, (1 << 27) // (HKV * case["rep"] * case["new"] * (case["vis"] + s["k_fp"].shape[2])))
    return [slice(b, min(b + step, case["batch"])) for b in range(0, case["batch"], step)]


def _scores(s, b):
    """Scores [requests, HKV, new * rep, vis + fp], keys in cache order [visual | system, text]; -inf where a key does not count."""
    case = s["case"]
    vis, t_fp, new = case["vis"], s["k_fp"].shape[2], case["new"]
    k = torch.cat([_unpack([t[b] for t in s["k_pack"]]), s["k_fp"][b].float().transpose(2, 3)], -1)      # [.., HKV, D, keys]
    q = s["q"][b].unflatten(2, (HKV, -1)).transpose(1, 2).flatten(2, 3).float()                           # [.., HKV, new * rep, D]
    sc = (q @ k) * (1 / math.sqrt(D))
    seen = torch.ones(new, 1, vis + t_fp, dtype=torch.bool, device=k.device)
    seen[:, 0, vis:] = torch.arange(t_fp, device=k.device) <= torch.arange(t_fp - new, t_fp, device=k.device).unsqueeze(1)
    seen = seen.expand(-1, case["rep"], -1).flatten(0, 1)
    if s["mask"] is not None:                                                # in key order [system | visual | text]
        m = s["mask"][b].float()
        m = torch.cat([m[:, SYS:SYS + vis], m[:, :SYS], m[:, SYS + vis:]], -1)[:, None, None]
        sc = sc + m
        seen = seen & (m != -math.inf)
    return torch.where(seen, sc, -math.inf)


def _plain_chunk(s):
    case, q = s["case"], s["q"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[0], q.shape[2], case["new"], device=q.device)
    for b in _requests(s):
        sc = _scores(s, b)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        v = torch.cat([_unpack([t[b] for t in s["v_pack"]]), s["v_fp"][b].float()], 2)
        o = (p @ v) / torch.where(total == 0, 1.0, total)
        out[b] = o.unflatten(2, (case["new"], -1)).transpose(1, 2).flatten(2, 3).to(q.dtype)
        lse[b] = (top + torch.log(total)).unflatten(2, (case["new"], -1)).squeeze(-1).transpose(2, 3).flatten(1, 2)
    return out, lse


def _plain_weights(s):
    case = s["case"]
    w = torch.empty(case["batch"], HKV, case["vis"] + s["k_fp"].shape[2], device=s["q"].device)
    for b in _requests(s):
        lse = s["lse"][b].unflatten(1, (HKV, -1)).transpose(2, 3).flatten(2).unsqueeze(-1)
        w[b] = torch.exp(_scores(s, b) - torch.where(lse == -math.inf, 0.0, lse)).sum(2)      # a row without keys: all of them -inf
    return w[..., :case["vis"]].contiguous(), w[..., case["vis"]:].contiguous()


def _largest(rank, keep):
    """Indices of the ``keep`` largest of the last dimension, ties to the lowest index, in ascending order."""
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    return order[..., :keep].sort(-1).values


def _plain_groups(s):
    keep, w = s["case"]["keep"], s["weights"].unflatten(-1, (-1, GROUP))
    kept = _largest(w.double().sum(-1), keep)                # in 64 bits: the sums decide a border
    (kc, ks, km), (vc, vs, vm) = s["k_pack"], s["v_pack"]

    def columns(t):                                          # [B,H,D,groups * n]
        n = t.shape[-1] // w.shape[2]
        t = t.unflatten(-1, (-1, n))
        return t.gather(3, kept[:, :, None, :, None].expand(-1, -1, D, -1, n)).flatten(-2)

    def tokens(t):                                           # [B,H,groups * 32,n]
        t = t.unflatten(2, (-1, GROUP))
        return t.gather(2, kept[..., None, None].expand(-1, -1, -1, GROUP, t.shape[-1])).flatten(2, 3)

    return (columns(kc), columns(ks), columns(km), tokens(vc), tokens(vs), tokens(vm),
            w.gather(2, kept[..., None].expand(-1, -1, -1, GROUP)).flatten(2), kept)


def _plain_tokens(s):
    case, w = s["case"], s["weights"]
    rank = w.clone()
    rank[..., :SYS] = math.inf
    rank[..., case["text"] - case["recent"]:] = math.inf
    kept = _largest(rank, case["keep"])
    row = kept.unsqueeze(-1).expand(-1, -1, -1, D)
    return s["k_fp"].gather(2, row), s["v_fp"].gather(2, row), w.gather(2, kept), kept


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"chunk": _plain_chunk, "weights": _plain_weights, "groups": _plain_groups, "tokens": _plain_tokens}[op](state)
    from calibquant_b200 import ops
    s, case = state, state["case"]
    if op == "chunk":
        return ops.chunk_attention(s["q"], s["k_pack"], s["v_pack"], s["k_fp"], s["v_fp"], SYS, mask=s["mask"], return_lse=True)
    if op == "weights":
        return ops.key_weights(s["q"], s["lse"], s["k_pack"], s["k_fp"], SYS, mask=s["mask"])
    if op == "groups":      # codes move as the words that hold them, so they are compared as whole numbers
        k_pack, v_pack, weights, kept = ops.evict_groups(s["k_pack"], s["v_pack"], s["weights"], case["keep"], bits=4)
        return (*k_pack, *v_pack, weights, kept)
    return ops.evict_tokens(s["k_fp"], s["v_fp"], s["weights"], case["keep"], t_sys=SYS, recent=case["recent"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    pairs, B = HKV * case["batch"], case["batch"]
    if case["op"] == "groups":
        n, kept = case["vis"], case["keep"] * GROUP
        return {"bytes": pairs * (4 * n + 2 * kept * 160 + 4 * kept + 8 * case["keep"]), "flops": pairs * n}
    if case["op"] == "tokens":
        n, kept = case["text"], case["keep"]
        return {"bytes": pairs * (4 * n + 2 * kept * 512 + 4 * kept + 8 * kept), "flops": pairs * n}
    new, vis, rep = case["new"], case["vis"], case["rep"]
    t_fp = SYS + case["text"] + new
    seen = new * (vis + t_fp - new) + new * (new + 1) // 2
    rows = pairs * rep * new
    mask = 2 * B * (vis + t_fp) if case["mask"] else 0
    if case["op"] == "chunk":
        return {"bytes": pairs * (160 * vis + 512 * t_fp) + rows * (512 + 4) + mask, "flops": 4 * D * pairs * rep * seen}
    return {"bytes": pairs * (80 * vis + 256 * t_fp + 4 * (vis + t_fp)) + rows * (256 + 4) + mask, "flops": 2 * D * pairs * rep * seen}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------
def _value64(pack):
    """scale * code + minimum, the codes taken from the bytes of the words."""
    code, scale, mn = pack
    byte = code.contiguous().view(torch.uint8)
    c = torch.empty(*byte.shape[:-1], byte.shape[-1] * 2, dtype=torch.float64, device=code.device)
    c[..., 0::2], c[..., 1::2] = byte % 16, byte // 16
    return c * scale.double().repeat_interleave(GROUP, -1) + mn.double().repeat_interleave(GROUP, -1)


def _attention64(s, b, head):
    """Scores of one query head against its keys [system | visual | text], and which of them take part."""
    case, h = s["case"], head // s["case"]["rep"]
    vis, new = case["vis"], case["new"]
    keys = s["k_fp"][b, h].double()
    keys = torch.cat([keys[:SYS], _value64([t[b, h] for t in s["k_pack"]]).T, keys[SYS:]])
    n = keys.shape[0]
    score = torch.einsum("id,kd->ik", s["q"][b, :, head].double(), keys) / D ** 0.5
    last = torch.arange(new, device=score.device)[:, None] + (n - new)
    hidden = torch.arange(n, device=score.device)[None, :] > last
    if s["mask"] is not None:
        hidden = hidden | torch.isneginf(s["mask"][b])[None, :]
        score = score + s["mask"][b].double()
    return score.masked_fill(hidden, -math.inf)


def exact(case, seed):
    s = prepare(case, seed)
    B, op = case["batch"], case["op"]
    if op == "chunk":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        lse = torch.empty(B, out.shape[2], case["new"], dtype=torch.float64, device=out.device)
        for b in range(B):
            for head in range(out.shape[2]):
                score, h = _attention64(s, b, head), head // case["rep"]
                v = s["v_fp"][b, h].double()
                v = torch.cat([v[:SYS], _value64([t[b, h] for t in s["v_pack"]]), v[SYS:]])
                lse[b, head] = torch.logsumexp(score, -1)
                out[b, :, head] = torch.exp(score - lse[b, head][:, None]).nan_to_num(0.0) @ v
        return out, lse
    if op == "weights":
        w = torch.zeros(B, HKV, case["vis"] + s["k_fp"].shape[2], dtype=torch.float64, device=s["q"].device)
        for b in range(B):
            for head in range(HKV * case["rep"]):
                p = torch.exp(_attention64(s, b, head) - s["lse"][b, head].double()[:, None])
                w[b, head // case["rep"]] += p.nan_to_num(0.0).sum(0)
        end = SYS + case["vis"]
        return w[..., SYS:end], torch.cat([w[..., :SYS], w[..., end:]], -1)
    # a selection has no computed numbers: the ranking by comparison of Python numbers, row by row
    unit = GROUP if op == "groups" else 1
    w = s["weights"].double().unflatten(-1, (-1, unit)).sum(-1)
    kept = torch.empty(B, HKV, case["keep"], dtype=torch.int64)
    for b in range(B):
        for h in range(HKV):
            row = w[b, h].tolist()
            n = len(row)
            if op == "tokens":
                row = [math.inf if t < SYS or t >= n - case["recent"] else x for t, x in enumerate(row)]
            kept[b, h] = torch.tensor(sorted(sorted(range(n), key=lambda t: (-row[t], t))[:case["keep"]]))
    kept = kept.to(w.device)
    bi = torch.arange(B, device=w.device)[:, None, None]
    hi = torch.arange(HKV, device=w.device)[None, :, None]
    token = (kept[..., None] * unit + torch.arange(unit, device=w.device)).flatten(2)
    if op == "tokens":
        return s["k_fp"][bi, hi, token], s["v_fp"][bi, hi, token], s["weights"][bi, hi, token], kept
    word = (kept[..., None] * 4 + torch.arange(4, device=w.device)).flatten(2)      # four words of eight tokens
    kc, ks, km = s["k_pack"]
    columns = [t.transpose(2, 3)[bi, hi, i].transpose(2, 3) for t, i in ((kc, word), (ks, kept), (km, kept))]
    return (*columns, *(t[bi, hi, token] for t in s["v_pack"]), s["weights"][bi, hi, token], kept)
