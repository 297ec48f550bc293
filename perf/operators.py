"""What is measured of the 4-bit key/value cache: appending to it, attending over it, the
attention weight that each cached token gathers, and eviction by that weight.

The cache holds K and V as MXFP4: packed E2M1 codes (element 2i in the low nibble) with one
UE8M0 scale byte (2^(byte - 127), bytes 67..192) per 32 channels, in pages of `page` tokens:

    k, v              uint8 [pages, kv_heads, page, dim / 2]
    k_scale, v_scale  uint8 [pages, kv_heads, page, dim / 32]

Sequence b's token j lies in page table[b, j // page], slot j % page; lens[b] counts its tokens,
the ones appended in this step (rows cu[b]..cu[b+1] of q, k, v) among them and last.
"""
import math

import torch

own = False

CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOW, HIGH = 67, 192  # scale bytes of the cache


# ----------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a serving batch stores one token for each sequence: latency counts
        dict(name="append_step", op="append", seqs=48, new=1, len=2048, kv_heads=8, dim=128, page=64, type="bf16"),
        # prompts of odd lengths are stored at once, from an fp32 projection
        dict(name="append_prompts", op="append", seqs=7, new=6001, len=6500, kv_heads=4, dim=64, page=16, type="f32"),
        # one user, one token, a short context: the smallest call
        dict(name="decode_one", op="attention", seqs=1, new=1, len=1777, heads=32, kv_heads=8, dim=128, page=64,
             window=0, softcap=0.0, causal=True),
        # a decode step of a batch with ragged contexts
        dict(name="decode_batch", op="attention", seqs=48, new=1, len=8192, heads=32, kv_heads=8, dim=128, page=64,
             window=0, softcap=0.0, causal=True),
        # a decode step over long contexts with few key/value heads
        dict(name="decode_long", op="attention", seqs=2, new=1, len=131072, heads=64, kv_heads=4, dim=128, page=128,
             window=0, softcap=0.0, causal=True),
        # a few drafted tokens are verified at once; capped scores, sliding window, seven heads to a group
        dict(name="verify_window", op="attention", seqs=20, new=4, len=7000, heads=28, kv_heads=4, dim=256, page=32,
             window=4096, softcap=50.0, causal=True),
        # a chunk of a long prompt over what is cached of it
        dict(name="prompt_chunk", op="attention", seqs=1, new=2048, len=16500, heads=32, kv_heads=8, dim=128, page=64,
             window=0, softcap=0.0, causal=True),
        # ragged prompts, whole
        dict(name="prompts_ragged", op="attention", seqs=5, new=1900, len=1900, heads=24, kv_heads=8, dim=64, page=16,
             window=0, softcap=30.0, causal=True),
        # the weight that one decode step gives each cached token
        dict(name="weights_step", op="weights", seqs=32, new=1, len=4096, heads=32, kv_heads=8, dim=128, page=64,
             window=0, softcap=0.0, causal=True),
        # the weight that the last tokens of a prompt give it, before the prompt's cache is thinned out
        dict(name="weights_prompt", op="weights", seqs=3, new=32, len=32000, heads=32, kv_heads=8, dim=128, page=64,
             window=0, softcap=0.0, causal=True),
        # one sequence over its budget
        dict(name="evict_one", op="evict", seqs=1, len=4500, budget=4096, sink=4, recent=64, kv_heads=8, dim=128, page=64),
        # a batch of ragged sequences is thinned out to a quarter
        dict(name="evict_batch", op="evict", seqs=24, len=8000, budget=2001, sink=4, recent=256, kv_heads=8, dim=128,
             page=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {o: [max(work(c)[k] for c in listed() if c["op"] == o) for k in ("bytes", "flops")]
            for o in ("append", "attention", "weights", "evict")}
    while True:
        op = rng.choice(("append", "attention", "attention", "attention", "weights", "evict"))
        kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 256))
        c = dict(op=op, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128)))
        if op == "append":
            new = rng.choice((1, _spread(rng, 1, 6001)))
            c |= dict(seqs=_spread(rng, 1, 64), new=new, len=new + _spread(rng, 1, 2048), type=rng.choice(("bf16", "f32")))
        elif op == "evict":
            length = _spread(rng, 300, 16000)
            budget = max(2, int(length * rng.uniform(0.1, 1.1)))
            sink = rng.randrange(0, min(8, budget))
            c |= dict(seqs=_spread(rng, 1, 48), len=length, budget=budget, sink=sink,
                      recent=rng.randrange(0, min(budget - sink, 512) + 1))
        else:
            form = rng.choice(("step", "draft", "prompt"))
            group = rng.choice((1, 2, 4, 5, 7, 8, 16))
            new = 1 if form == "step" else rng.randrange(2, 9) if form == "draft" else _spread(rng, 16, 2048)
            length = new + _spread(rng, 1, 131072 if form == "step" else 16000)
            if op == "weights":
                new = min(new, 64)
            c |= dict(seqs=_spread(rng, 1, 64 if form != "prompt" else 8), new=new, len=length, heads=kv_heads * group,
                      window=rng.choice((0, 0, _spread(rng, 64, 8192))), softcap=rng.choice((0.0, 0.0, 30.0, 50.0)),
                      causal=rng.choice((True, True, True, False)))
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _rows(c) <= _rows(dict(listed()[6])):
            return c


def _rows(c):
    """Scores, padded: what the plain form holds of a case."""
    return c["seqs"] * c.get("heads", 0) * c.get("new", 0) * c["len"]


def _sizes(c):
    """(new tokens, length) of each sequence: the first as the case says, the others spread below."""
    got = []
    for b in range(c["seqs"]):
        part = 1.0 if b == 0 else 0.25 + 0.75 * ((b * 0.6180339887) % 1.0)
        new = max(1, int(c.get("new", 0) * part)) if "new" in c else 0
        got.append((new, max(new, int(c["len"] * part))))
    return got


def _seen(c, new, length):
    """(cached tokens that some query sees, pairs of query and token) of a sequence."""
    lo = min(max(0, length - new + 1 - c["window"]), length) if c["window"] else 0
    pairs = 0
    for i in range(new):
        at = length - new + i
        end = at + 1 if c["causal"] else length
        pairs += end - (max(0, at + 1 - c["window"]) if c["window"] else 0)
    return length - lo, pairs


def work(c):
    sizes, heads = _sizes(c), c["kv_heads"]
    token = heads * (c["dim"] // 2 + c["dim"] // 32)  # bytes of K, or V, of one cached token
    if c["op"] == "append":
        rows = sum(n for n, _ in sizes)
        return {"bytes": rows * (heads * c["dim"] * 2 * (4 if c["type"] == "f32" else 2) + 2 * token + heads * c["dim"] * 4),
                "flops": 0}
    if c["op"] == "evict":
        kept = sum(min(n, c["budget"]) for _, n in sizes)
        return {"bytes": 4 * heads * sum(n for _, n in sizes) + kept * (2 * 2 * token + heads * (4 + 4 + c["dim"] * 4)),
                "flops": 0}
    seen = [_seen(c, *s) for s in sizes]
    rows, tokens, pairs = sum(n for n, _ in sizes) * c["heads"], sum(s for s, _ in seen), sum(p for _, p in seen)
    if c["op"] == "attention":
        return {"bytes": tokens * 2 * token + rows * (4 * c["dim"] + 4), "flops": 4 * c["dim"] * c["heads"] * pairs}
    return {"bytes": tokens * (token + 8 * heads) + rows * (2 * c["dim"] + 4), "flops": 2 * c["dim"] * c["heads"] * pairs}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    sizes = _sizes(c)
    news, lens = [n for n, _ in sizes], [n for _, n in sizes]
    width = -(-max(lens) // c["page"])
    out_width = -(-c["budget"] // c["page"]) if c["op"] == "evict" else 0
    pages = c["seqs"] * (width + out_width)
    shape = (pages, c["kv_heads"], c["page"])
    at = torch.randperm(pages, generator=gen, device=dev).to(torch.int32).view(c["seqs"], width + out_width)
    s = dict(case=c, table=at[:, :width].contiguous(), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
             longest=max(lens))
    # keys have channels that are larger than the others throughout, values have not
    channel = torch.exp(0.7 * torch.randn(c["kv_heads"], 1, c["dim"], generator=gen, device=dev))
    for name, by in (("k", channel), ("v", None)):
        codes = torch.empty((*shape, c["dim"] // 2), dtype=torch.uint8, device=dev)
        scale = torch.empty((*shape, c["dim"] // 32), dtype=torch.uint8, device=dev)
        step = max(1, (1 << 26) // (c["kv_heads"] * c["page"] * c["dim"]))
        for p in range(0, pages, step):
            x = torch.randn((min(step, pages - p), *shape[1:], c["dim"]), generator=gen, device=dev)
            codes[p:p + step], scale[p:p + step] = _quantise(x if by is None else x * by)
        s[name], s[name + "_scale"] = codes, scale
    if c["op"] == "evict":
        s["out_table"] = at[:, width:].contiguous()
        # what tokens gather is spread over orders of magnitude, and some gather nothing
        w = torch.exp(2.5 * torch.randn(shape, generator=gen, device=dev))
        s["weights"] = torch.where(torch.rand(shape, generator=gen, device=dev) < 0.03, torch.zeros_like(w), w)
        kept = [min(n, c["budget"]) for n in lens]
        s["cu"] = torch.tensor([0, *kept], dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)
        s["start"], s["rows"] = torch.zeros(c["seqs"], dtype=torch.int32, device=dev), sum(kept)
        return s
    rows = sum(news)
    s["cu"] = torch.tensor([0, *news], dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)
    s["rows"] = rows
    if c["op"] == "append":
        kind = torch.float32 if c["type"] == "f32" else torch.bfloat16
        new = torch.randn((rows, 2, c["kv_heads"], c["dim"]), generator=gen, device=dev)
        new[:, 0] *= channel[:, 0]
        s["new_k"], s["new_v"] = new.to(kind).unbind(1)  # both are parts of one projection's rows
        s["start"] = s["lens"] - torch.tensor(news, dtype=torch.int32, device=dev)
        return s
    q = torch.randn((rows, c["heads"] + 2 * c["kv_heads"], c["dim"]), generator=gen, device=dev)
    s["q"] = q.to(torch.bfloat16)[:, :c["heads"]]  # a part of one projection's rows
    s["scale"] = 1.0 / math.sqrt(c["dim"])
    if c["op"] == "weights":
        s["lse"] = _lse(s)
        s["weights"] = torch.rand(shape, generator=gen, device=dev)
        s["sums"] = torch.zeros(shape, device=dev)
    return s


# ----------------------------------------------------------------- the operators, as a user calls them or in their plain form
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"append": _append, "attention": _attention, "weights": _weights, "evict": _evict}[op](state)


def _own(s, op):
    from gcnasm_b200 import kv4

    c = s["case"]
    cache = kv4.KV4Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "append":
        kv4.append(cache, s["new_k"], s["new_v"], s["table"], s["lens"], s["cu"], max_new=c["new"])
        return kv4.read(cache, s["table"], s["start"], s["cu"], s["rows"])
    if op == "evict":
        kept, lens = kv4.evict(cache, s["weights"], s["table"], s["lens"], c["budget"], sink=c["sink"], recent=c["recent"],
                               out_table=s["out_table"])
        k, v = kv4.read(cache, s["out_table"], s["start"], s["cu"], s["rows"])
        return {"kept": kept, "lens": lens, "weights": s["weights"], "k": k, "v": v}
    mask = dict(scale=s["scale"], causal=c["causal"], window=c["window"], softcap=c["softcap"], max_q=c["new"])
    cu = s["cu"] if c["new"] > 1 else None
    if op == "attention":
        return kv4.attention(s["q"], cache, s["table"], s["lens"], cu, **mask)
    return kv4.weights(s["q"], s["lse"], cache, s["table"], s["lens"], s["weights"], cu, out=s["sums"], **mask)


def _quantise(x):
    """fp32 [..., dim] -> (packed codes, scale bytes): the least power of two s with 6 s >= the block's
    largest magnitude, and the nearest code of x / s, a tie to the even code."""
    blocks = x.unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1)
    part, power = torch.frexp(largest)
    byte = (torch.where(part <= 0.75, power - 3, power - 2) + 127).clamp(LOW, HIGH)
    y = (blocks * torch.exp2(127.0 - byte).unsqueeze(-1)).flatten(-2)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + 8 * (y < 0)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _values(codes, scale):
    """Packed codes and scale bytes -> fp32."""
    table = torch.tensor(CODES + tuple(-v for v in CODES), device=codes.device)
    both = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    return (both.unflatten(-1, (-1, 32)) * torch.exp2(scale.clamp(LOW, HIGH).float() - 127.0).unsqueeze(-1)).flatten(-2)


def _place(s, table, tokens, of):
    """Page and slot of tokens `tokens` of sequences `of`."""
    page = s["case"]["page"]
    return table[of, tokens // page].long(), tokens % page


def _new_rows(s):
    """Sequence and token of each of the rows cu[b]..cu[b+1]."""
    row = torch.arange(s["rows"], device=s["cu"].device)
    of = torch.searchsorted(s["cu"][1:].contiguous(), row, right=True)
    return of, s["start"][of].long() + row - s["cu"][of]


def _read(s, table):
    of, token = _new_rows(s)
    page, slot = _place(s, table, token, of)
    return tuple(_values(s[n][page, :, slot], s[n + "_scale"][page, :, slot]).to(torch.bfloat16) for n in ("k", "v"))


def _append(s):
    of, token = _new_rows(s)
    page, slot = _place(s, s["table"], token, of)
    for name, x in (("k", s["new_k"]), ("v", s["new_v"])):
        s[name][page, :, slot], s[name + "_scale"][page, :, slot] = _quantise(x.float())
    return _read(s, s["table"])


def _cached(s, name):
    """fp32 [seqs, kv_heads, longest, dim] of all that is cached."""
    c = s["case"]
    token = torch.arange(s["longest"], device=s["cu"].device).expand(c["seqs"], -1)
    page, slot = _place(s, s["table"], token, torch.arange(c["seqs"], device=token.device).unsqueeze(1))
    return _values(s[name][page, :, slot], s[name + "_scale"][page, :, slot]).transpose(1, 2)


def _scores(s):
    """(scores [seqs, kv_heads, new, group, longest] in fp32 with -inf where a query does not look, whether a
    row [seqs, new] is there, its row of q)."""
    c, dev = s["case"], s["cu"].device
    group = c["heads"] // c["kv_heads"]
    i = torch.arange(c["new"], device=dev)
    new = (s["cu"][1:] - s["cu"][:-1]).unsqueeze(1)
    there = i < new
    row = (s["cu"][:-1].unsqueeze(1) + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().unflatten(2, (c["kv_heads"], group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = (q @ _cached(s, "k").transpose(2, 3) * s["scale"]).unflatten(2, (c["new"], group))
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    at = (s["lens"].unsqueeze(1) - new + i).unsqueeze(-1)
    token = torch.arange(s["longest"], device=dev)
    sees = (token < s["lens"][:, None, None]) & there.unsqueeze(-1)
    if c["causal"]:
        sees = sees & (token <= at)
    if c["window"]:
        sees = sees & (token > at - c["window"])
    return score.masked_fill(~sees[:, None, :, None], -math.inf), there, row


def _attention(s):
    score, there, _ = _scores(s)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)  # a row that looks at nothing has no score
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ _cached(s, "v")).unflatten(2, score.shape[2:4]) / total.clamp(min=1e-30)
    lse = (top + torch.log(total)).squeeze(-1)
    out = out.permute(0, 2, 1, 3, 4)[there].flatten(1, 2)
    return out.to(torch.bfloat16), lse.permute(0, 2, 1, 3)[there].flatten(1, 2)


def _lse(s):
    return _attention(s)[1]


def _weights(s):
    c = s["case"]
    score, there, row = _scores(s)
    lse = s["lse"][row].unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 1, 3).unsqueeze(-1)
    gathered = torch.exp(score - lse.clamp(min=-1e30)).sum((2, 3))
    token = torch.arange(s["longest"], device=row.device).expand(c["seqs"], -1)
    of = torch.arange(c["seqs"], device=row.device).unsqueeze(1).expand_as(token)
    there = token < s["lens"].unsqueeze(1)
    of, token = of[there], token[there]
    page, slot = _place(s, s["table"], token, of)
    s["sums"][page, :, slot] = s["weights"][page, :, slot] + gathered[of, :, token]
    return s["sums"]


def _evict(s):
    c, dev = s["case"], s["cu"].device
    lens = s["lens"].unsqueeze(1)
    token = torch.arange(s["longest"], device=dev).expand(c["seqs"], -1)
    of = torch.arange(c["seqs"], device=dev).unsqueeze(1)
    page, slot = _place(s, s["table"], token, of)
    held = s["weights"][page, :, slot]  # [seqs, longest, kv_heads]
    # what is always kept ranks above every weight, what is not there below
    always = (token < c["sink"]) | (token >= lens - c["recent"])
    rank = torch.where(always.unsqueeze(-1), torch.full_like(held, math.inf), held)
    rank = torch.where((token < lens).unsqueeze(-1), rank, torch.full_like(held, -math.inf)).transpose(1, 2)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    kept = torch.nn.functional.pad(kept, (0, c["budget"] - kept.shape[-1]), value=s["longest"])
    new_lens = s["lens"].clamp(max=c["budget"])
    there = torch.arange(c["budget"], device=dev) < new_lens[:, None, None]
    kept = torch.sort(torch.where(there, kept, torch.full_like(kept, s["longest"])), dim=-1).values
    b, h, i = there.expand_as(kept).nonzero().unbind(1)
    page, slot = _place(s, s["table"], kept[b, h, i], b)
    to_page, to_slot = _place(s, s["out_table"], i, b)
    for name in ("k", "v", "k_scale", "v_scale", "weights"):
        s[name][to_page, h, to_slot] = s[name][page, h, slot]
    k, v = _read(s, s["out_table"])
    kept = torch.where(there, kept, torch.full_like(kept, -1)).to(torch.int32)
    return {"kept": kept, "lens": new_lens, "weights": s["weights"], "k": k, "v": v}


# ----------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](s)


def _exact_value(byte, scale, odd):
    code = (byte.long() >> (4 * odd)) & 15
    e, m = (code >> 1) & 3, (code & 1).double()
    size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double()))
    return torch.where(code >= 8, -size, size) * torch.exp2(scale.double() - 127)


def _exact_tokens(s, name, table, b, tokens):
    """float64 [tokens, kv_heads, dim] of one sequence."""
    page, slot = table[b].long()[tokens // s["case"]["page"]], tokens % s["case"]["page"]
    codes, scale = s[name][page, :, slot], s[name + "_scale"][page, :, slot].repeat_interleave(16, dim=-1)
    out = torch.empty((*codes.shape[:2], s["case"]["dim"]), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = _exact_value(codes, scale, 0), _exact_value(codes, scale, 1)
    return out


def _exact_append(s):
    def stored(x):
        y = x.double().unflatten(-1, (-1, 32))
        power = torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True) / 6)).clamp(LOW - 127, HIGH - 127)
        y = y / torch.exp2(power)
        a = y.abs()  # the grid's step is a half below 2, one below 4, two above; a tie goes to the even multiple
        a = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2))).clamp(max=6)
        return (torch.sign(y) * a * torch.exp2(power)).flatten(-2)

    return stored(s["new_k"]), stored(s["new_v"])


def _exact_rows(s, of_head):
    """Calls of_head(b, h, first row, scores [new, group, len]) for each sequence and key/value head, scores in 64 bits."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b in range(c["seqs"]):
        token = torch.arange(lens[b], device=s["cu"].device)
        k = _exact_tokens(s, "k", s["table"], b, token)
        at = lens[b] - (cu[b + 1] - cu[b]) + torch.arange(cu[b + 1] - cu[b], device=token.device).unsqueeze(1)
        hidden = torch.zeros((at.shape[0], lens[b]), dtype=torch.bool, device=token.device)
        if c["causal"]:
            hidden |= token > at
        if c["window"]:
            hidden |= token <= at - c["window"]
        for h in range(c["kv_heads"]):
            score = torch.einsum("igd,td->igt", s["q"][cu[b]:cu[b + 1], h * group:(h + 1) * group].double(), k[:, h]) / math.sqrt(c["dim"])
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            of_head(b, h, cu[b], score.masked_fill(hidden.unsqueeze(1), -math.inf))


def _exact_attention(s):
    c, token = s["case"], torch.arange(s["longest"], device=s["cu"].device)
    group, lens = c["heads"] // c["kv_heads"], s["lens"].tolist()
    out = torch.zeros((s["rows"], c["heads"], c["dim"]), dtype=torch.float64, device=token.device)
    lse = torch.zeros((s["rows"], c["heads"]), dtype=torch.float64, device=token.device)

    values = {}  # of the sequence that is at hand

    def of_head(b, h, row, score):
        if b not in values:
            values.clear()
            values[b] = _exact_tokens(s, "v", s["table"], b, token[:lens[b]])
        at = slice(row, row + score.shape[0]), slice(h * group, (h + 1) * group)
        lse[at] = torch.logsumexp(score, -1)
        out[at] = torch.einsum("igt,td->igd", torch.softmax(score, -1), values[b][:, h])

    _exact_rows(s, of_head)
    return out, lse


def _exact_weights(s):
    c = s["case"]
    group, page = c["heads"] // c["kv_heads"], c["page"]
    sums = s["sums"].double()

    def of_head(b, h, row, score):
        lse = s["lse"][row:row + score.shape[0], h * group:(h + 1) * group].double()
        token = torch.arange(score.shape[-1], device=score.device)
        at = s["table"][b].long()[token // page], h, token % page
        sums[at] = s["weights"][at].double() + torch.exp(score - lse.unsqueeze(-1)).sum((0, 1))

    _exact_rows(s, of_head)
    return sums


def _exact_evict(s):
    c, page = s["case"], s["case"]["page"]
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    dev = s["cu"].device
    weights = s["weights"].double()
    k = torch.empty((s["rows"], c["kv_heads"], c["dim"]), dtype=torch.float64, device=dev)
    v = torch.empty_like(k)
    kept = torch.full((c["seqs"], c["kv_heads"], c["budget"]), -1, dtype=torch.int32, device=dev)
    for b in range(c["seqs"]):
        token = torch.arange(lens[b], device=dev)
        ks, vs = _exact_tokens(s, "k", s["table"], b, token), _exact_tokens(s, "v", s["table"], b, token)
        n = min(lens[b], c["budget"])
        for h in range(c["kv_heads"]):
            w = s["weights"][s["table"][b].long()[token // page], h, token % page].double()
            w[:c["sink"]] = math.inf
            w[max(0, lens[b] - c["recent"]):] = math.inf
            order = torch.argsort(-w, stable=True)
            keep = torch.sort(order[:n]).values
            kept[b, h, :n] = keep.int()
            k[cu[b]:cu[b + 1], h], v[cu[b]:cu[b + 1], h] = ks[keep, h], vs[keep, h]
            to = torch.arange(n, device=dev)
            weights[s["out_table"][b].long()[to // page], h, to % page] = \
                s["weights"][s["table"][b].long()[keep // page], h, keep % page].double()
    return {"kept": kept, "lens": s["lens"].clamp(max=c["budget"]), "weights": weights, "k": k, "v": v}
