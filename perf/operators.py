"""Operators of a paged cache of keys and values, measured through gpt_b200.Backend.

Three families, each over its own range of sizes:

  write    new rows of keys and values go into the pages of their sequences, as they are or in 8 bits (e4m3 codes with a power of two
           for each token and head)
  read     rows come back out of the pages
  attend   attention of new tokens over the pages: single tokens, portions of prompts, whole prompts; all keys up to a token's own
           position, or a window of the last ones and a few first ones

The cache is [page][keys, values][key / value head][token of the page][dimension]; a sequence's pages are in its row of a table.  The
new rows of all sequences lie one behind the other; `lengths` counts a sequence's tokens with its new ones, so that the last new row
is the token at position length - 1.  A case is a dict of plain values; see listed() for the fixed ones and draw() for the ranges.
"""
import math

import torch

own = False

E4M3_MOST = 448.0          # largest value of a code
EXPONENTS = (-117, 119)    # of a row's power of two: every code times it is zero or a normal fp32 and bf16 value


def listed():
    return [
        # uneven prompts' keys and values on their way into an 8-bit cache (a layer of 8 key / value heads of 128)
        dict(name="write_prompts_e4m3", kind="write", sequences=12, new=4096, context=4096, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", cache="e4m3"),
        # one decoding step of 64 sequences: a row each
        dict(name="write_tokens_e4m3", kind="write", sequences=64, new=1, context=512, heads=12, kv_heads=4, dim=64, page=16, dtype="bf16", cache="e4m3"),
        # sequences on their way out of an 8-bit cache, to be kept elsewhere
        dict(name="read_e4m3", kind="read", sequences=6, new=8192, context=8192, heads=16, kv_heads=4, dim=128, page=64, dtype="bf16", cache="e4m3"),
        # a text of GPT-2's length
        dict(name="read_text_f32", kind="read", sequences=1, new=256, context=256, heads=12, kv_heads=12, dim=64, page=16, dtype="f32", cache="f32"),
        # one user's next token, GPT-2's heads
        dict(name="token_f32", kind="attend", sequences=1, new=1, context=256, heads=12, kv_heads=12, dim=64, page=16, dtype="f32", cache="f32", cap=0.0, window=0, sinks=0),
        # GPT-2's prompts
        dict(name="prompts_f32", kind="attend", sequences=8, new=256, context=256, heads=12, kv_heads=12, dim=64, page=16, dtype="f32", cache="f32", cap=0.0, window=0, sinks=0),
        # a full batch of requests, a token each
        dict(name="tokens_bf16", kind="attend", sequences=64, new=1, context=4096, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache="bf16", cap=0.0, window=0, sinks=0),
        # a few very long sequences, a token each, capped scores
        dict(name="tokens_e4m3_long", kind="attend", sequences=4, new=1, context=65536, heads=16, kv_heads=4, dim=128, page=64, dtype="bf16", cache="e4m3", cap=40.0, window=0, sinks=0),
        # a batch that sees the last thousand tokens and the first four
        dict(name="tokens_window_e4m3", kind="attend", sequences=48, new=1, context=16384, heads=32, kv_heads=8, dim=128, page=32, dtype="bf16", cache="e4m3", cap=0.0, window=1024, sinks=4),
        # one whole prompt
        dict(name="prompt_bf16", kind="attend", sequences=1, new=8192, context=8192, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", cache="bf16", cap=0.0, window=0, sinks=0),
        # the next portions of long prompts
        dict(name="portions_e4m3", kind="attend", sequences=3, new=1000, context=16384, heads=16, kv_heads=4, dim=128, page=64, dtype="bf16", cache="e4m3", cap=0.0, window=0, sinks=0),
        # a prompt that sees the last thousand tokens and the first four, capped scores
        dict(name="prompt_window", kind="attend", sequences=1, new=8192, context=8192, heads=12, kv_heads=4, dim=64, page=128, dtype="bf16", cache="bf16", cap=40.0, window=1024, sinks=4),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        kind = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        c = dict(kind=kind, sequences=_log(rng, 1, 96), heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads, dim=rng.choice([64, 128, 128, 40, 80, 96, 32]),
                 page=rng.choice([8, 16, 32, 64, 128, 256]), dtype=dtype, cache=rng.choice([dtype, "e4m3"]), context=_log(rng, 16, 65536))
        c["new"] = {"write": rng.choice([1, _log(rng, 1, c["context"])]), "read": c["context"], "attend": rng.choice([1, 1, min(c["context"], _log(rng, 2, 8)), _log(rng, 1, min(c["context"], 8192))])}[kind]
        if kind == "attend":
            c["cap"] = rng.choice([0.0, 0.0, 0.0, 40.0])
            c["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
            c["sinks"] = rng.choice([0, 4, _log(rng, 1, 64)]) if c["window"] else 0
        tokens = c["sequences"] * c["context"] * c["kv_heads"] * c["dim"]
        scores = c["sequences"] * c["new"] * c["context"] * c["heads"]
        if tokens <= (1 << 28) and (kind != "attend" or scores * c["dim"] <= (1 << 38) / (8 if dtype == "f32" else 1)) and scores <= 1 << 31:
            return c


# ---- sizes of the sequences: the longest is `context` tokens, the others down to a quarter of it; `new` alike where it is more than a few


def _sizes(c):
    rng = _Counter(c["sequences"] * 7919 + c["context"] * 31 + c["new"])
    lengths, news = [], []
    for i in range(c["sequences"]):
        length = c["context"] if i == 0 else max(1, int(c["context"] * (0.25 + 0.75 * rng.next())))
        new = length if c["new"] == c["context"] else c["new"] if c["new"] == 1 or i == 0 else max(1, int(c["new"] * (0.25 + 0.75 * rng.next())))
        lengths.append(length)
        news.append(min(new, length))
    return lengths, news


class _Counter:
    """A few numbers in [0, 1) that go by the case alone: work() needs them without a device."""

    def __init__(self, seed):
        self.x = seed & 0x7FFFFFFF

    def next(self):
        self.x = (self.x * 1103515245 + 12345) & 0x7FFFFFFF
        return (self.x >> 8) / float(1 << 23)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths, news = _sizes(c)
    S, G, d, page = c["sequences"], c["kv_heads"], c["dim"], c["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")[:sum(counts)].to(torch.int32).cpu()
    table, at = torch.zeros(S, max(counts), dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    starts = torch.zeros(S + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(news, dtype=torch.int32).cumsum(0)
    rows = int(starts[-1])
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}
    s = dict(case=c, rows=rows, starts=starts.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), table=table.cuda(), most_new=max(news), longest=max(lengths))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    # tokens' keys and values differ in size, as a projection's do
    held = normal(pages, 2, G, page, d) * torch.exp(0.7 * normal(pages, 2, G, page, 1))
    if c["cache"] == "e4m3":
        codes, exponents = _codes(held)
        s["data"], s["scales"] = codes, exponents
    else:
        s["data"], s["scales"] = held.to(dt[c["cache"]]), None
    del held
    if c["kind"] == "write":
        kv = normal(rows, 2, G * d) * torch.exp(0.7 * normal(rows, 2, 1))
        s["k"], s["v"] = (kv[:, i].to(dt[c["dtype"]]).contiguous() for i in (0, 1))
    elif c["kind"] == "read":
        s["k"], s["v"] = (torch.empty(rows, G * d, device="cuda", dtype=dt[c["dtype"]]) for _ in (0, 1))
    else:
        s["q"] = normal(rows, c["heads"] * d).to(dt[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- the plain forms


def _codes(x):
    """e4m3 codes and one exponent (plus 127, a byte) for each last dimension of x, fp32."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))   # most = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)      # the smallest e with most <= 448 * 2^e = 0.875 * 2^(9 + e)
    e = torch.where(mantissa == 0, EXPONENTS[0], e).clamp(*EXPONENTS)
    codes = torch.ldexp(x, -e).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).squeeze(-1)


def _positions(s):
    """Sequence, position and index among its sequence's new rows of every row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    nth = row - s["starts"].long()[seq]
    new = (s["starts"][1:] - s["starts"][:-1]).long()[seq]
    return seq, s["lengths"].long()[seq] - new + nth, nth


def _places(s, seq, position):
    page = s["case"]["page"]
    return s["table"].long()[seq, position // page], position % page


def _held(s, data, which, where, token):
    """Keys (0) or values (1) of tokens in fp32: [..., kv_heads, dim]."""
    got = data[where, which, :, token]
    if s["scales"] is None:
        return got.float()
    return torch.ldexp(got.float(), s["scales"][where, which, :, token].int().unsqueeze(-1) - 127)


def _write(s):
    c = s["case"]
    seq, position, _ = _positions(s)
    where, token = _places(s, seq, position)
    data = s["data"].view(torch.uint8) if c["cache"] == "e4m3" else s["data"]
    for which, rows in ((0, s["k"]), (1, s["v"])):
        x = rows.float().view(s["rows"], c["kv_heads"], c["dim"])
        if c["cache"] == "e4m3":
            codes, exponents = _codes(x)
            data[where, which, :, token] = codes.view(torch.uint8)
            s["scales"][where, which, :, token] = exponents
        else:
            data[where, which, :, token] = x.to(data.dtype)


def _read(s):
    seq, position, _ = _positions(s)
    where, token = _places(s, seq, position)
    data = s["data"]
    for which, rows in ((0, s["k"]), (1, s["v"])):
        rows.copy_(_held(s, data, which, where, token).reshape(rows.shape))


def _attend(s):
    """All sequences side by side, padded to the most new rows and the longest sequence."""
    c = s["case"]
    S, H, G, d, N, L = c["sequences"], c["heads"], c["kv_heads"], c["dim"], s["most_new"], s["longest"]
    seq, _, nth = _positions(s)
    q = torch.zeros(S, N, H, d, device="cuda")
    q[seq, nth] = s["q"].float().view(-1, H, d)
    q = q.view(S, N, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * N, d)
    at = torch.arange(L, device="cuda").clamp(max=c["page"] * s["table"].shape[1] - 1)
    where, token = s["table"].long()[:, at // c["page"]], (at % c["page"]).expand(S, L)
    k, v = (_held(s, s["data"], which, where, token).transpose(1, 2) for which in (0, 1))   # [S, G, L, d]
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5)
    if c["cap"]:
        scores.div_(c["cap"]).tanh_().mul_(c["cap"])
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    own_position = ((s["lengths"].long() - new).unsqueeze(1) + torch.arange(N, device="cuda")).unsqueeze(2)   # [S, N, 1]
    hidden = at > own_position
    if c["window"]:
        hidden |= (own_position - at >= c["window"]) & (at >= c["sinks"])
    scores.view(S, G, H // G, N, L).masked_fill_(hidden.view(S, 1, 1, N, L), float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, v).div_(total)
    out = out.view(S, G, H // G, N, d).permute(0, 3, 1, 2, 4).reshape(S, N, H * d)
    s["out"].copy_(out[seq, nth])


# ---- the framework's calls

_backend = None


def _own(s):
    global _backend
    import gpt_b200
    if _backend is None:
        _backend = gpt_b200.Backend(0, torch.cuda.current_stream().cuda_stream)
    c = s["case"]
    if "pages" not in s:   # what a program keeps beside its cache and its batch
        s["pages"] = gpt_b200.KvPages(s["data"], s["scales"], {"bf16": gpt_b200.KV_BF16, "f32": gpt_b200.KV_F32, "e4m3": gpt_b200.KV_E4M3}[c["cache"]], s["data"].shape[0], c["page"], c["kv_heads"], c["dim"])
        s["batch"] = gpt_b200.KvRows(s["starts"], s["lengths"], s["table"], c["sequences"], s["table"].shape[1], s["rows"], s["most_new"])
    dtype = {"bf16": gpt_b200.DTYPE_BF16, "f32": gpt_b200.DTYPE_F32}[c["dtype"]]
    if c["kind"] == "write":
        _backend.kv_pages_write(s["pages"], s["batch"], s["k"], s["k"].shape[1], s["v"], s["v"].shape[1], dtype)
    elif c["kind"] == "read":
        _backend.kv_pages_read(s["k"], s["k"].shape[1], s["v"], s["v"].shape[1], dtype, s["pages"], s["batch"])
    else:
        _backend.attention_paged(s["out"], s["out"].shape[1], None, s["q"], s["q"].shape[1], dtype, c["heads"], s["pages"], s["batch"], c["dim"] ** -0.5, c["cap"], c["window"], c["sinks"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        _own(state)
    else:
        {"write": _write, "read": _read, "attend": _attend}[kind](state)
    if kind == "write":
        return {"data": state["data"], "scales": state["scales"]} if state["scales"] is not None else {"data": state["data"]}
    if kind == "read":
        return {"k": state["k"], "v": state["v"]}
    return {"out": state["out"]}


def _visible(c, length, new):
    """(query, key) pairs that see one another, and keys that any of the new tokens sees."""
    first = length - new
    if not c["window"]:
        return sum_to(length) - sum_to(first), length
    w, k = c["window"], c["sinks"]
    pairs = 0
    for p in range(first, length):
        low = max(0, p - w + 1)
        pairs += p - low + 1 + min(k, low)
    low = max(0, first - w + 1)
    return pairs, length - low + min(k, low)


def sum_to(n):
    return n * (n + 1) // 2


def work(case):
    c = dict(case)
    lengths, news = _sizes(c)
    rows, width = sum(news), 2 * c["kv_heads"] * c["dim"]
    size = {"bf16": 2, "f32": 4}[c["dtype"]]
    token = width * {"bf16": 2, "f32": 4, "e4m3": 1}[c["cache"]] + (2 * c["kv_heads"] if c["cache"] == "e4m3" else 0)
    if c["kind"] != "attend":
        return {"bytes": rows * (width * size + token), "flops": 0}
    pairs, keys = (sum(x) for x in zip(*(_visible(c, n, m) for n, m in zip(lengths, news))))
    return {"bytes": 2 * rows * c["heads"] * c["dim"] * size + keys * token, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- the same in 64 bits, from the definitions: sequence by sequence, head by head


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    lengths, news = _sizes(c)
    G, d, page = c["kv_heads"], c["dim"], c["page"]
    table = s["table"].cpu()
    at = 0
    results = []
    data = s["data"].double() if c["kind"] == "write" else s["data"]
    scales = s["scales"].clone() if s["scales"] is not None else None
    for i, (length, new) in enumerate(zip(lengths, news)):
        count = -(-length // page)
        ids = table[i, :count].long().cuda()
        if c["kind"] == "write":
            positions = torch.arange(length - new, length, device="cuda")
            where, token = ids[positions // page], positions % page
            for which, rows in ((0, s["k"]), (1, s["v"])):
                x = rows[at:at + new].double().reshape(new, G, d)
                if c["cache"] == "e4m3":
                    most = x.abs().amax(-1)
                    e = torch.ceil(torch.log2((most / 448.0).clamp(min=2.0 ** -140)))
                    e = torch.where(448.0 * torch.exp2(e - 1) >= most, e - 1, e)   # log2's rounding
                    e = torch.where(448.0 * torch.exp2(e) < most, e + 1, e).clamp(*EXPONENTS)
                    y = x / torch.exp2(e)[..., None]
                    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # three bits of mantissa, smallest normal 2^-6
                    data[where, which, :, token] = (torch.round(y / step) * step).clamp(-448.0, 448.0)
                    scales[where, which, :, token] = (e + 127).to(torch.uint8)
                else:
                    data[where, which, :, token] = x.to(s["data"].dtype).double()
        else:
            held = data[ids].double()   # [pages, 2, G, page, d]
            if scales is not None:
                held *= torch.exp2(scales[ids].double() - 127.0)[..., None]
            k, v = (held[:, which].permute(1, 0, 2, 3).reshape(G, count * page, d)[:, :length] for which in (0, 1))
            if c["kind"] == "read":
                results.append([x[:, length - new:].permute(1, 0, 2).reshape(new, G * d) for x in (k, v)])
            else:
                q = s["q"][at:at + new].double().reshape(new, c["heads"], d)
                out = torch.empty_like(q)
                key = torch.arange(length, device="cuda")
                mine = torch.arange(length - new, length, device="cuda")[:, None]
                seen = key <= mine
                if c["window"]:
                    seen &= (mine - key < c["window"]) | (key < c["sinks"])
                for h in range(c["heads"]):
                    g = h // (c["heads"] // G)
                    x = q[:, h] @ k[g].T / math.sqrt(d)
                    if c["cap"]:
                        x = c["cap"] * torch.tanh(x / c["cap"])
                    out[:, h] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ v[g]
                results.append(out.reshape(new, -1))
        at += new
    if c["kind"] == "write":
        return {"data": data, "scales": scales} if scales is not None else {"data": data}
    if c["kind"] == "read":
        return dict(zip("kv", (torch.cat(x) for x in zip(*results))))
    return {"out": torch.cat(results)}
