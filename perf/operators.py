"""The serving operators over a paged key/value cache, as cases that can be timed and compared: appending and reading the cache, attention of
new tokens over it, and what is done to logits before a token is chosen.

Four kinds of case:

  append   serving.kv_append: keys and values of new tokens, views of a fused projection, go to their pages (bf16, or e4m3 with a scale per row)
  read     serving.kv_read: whole contexts come back out of their pages as bf16 rows
  attend   serving.paged_attention: a chunk of new tokens per sequence, one token or thousands, attends over its pages
  logits   serving.logits_process: penalties of repeated tokens, biases and a grammar's bit mask

With `own` false, run() computes the operators in elementary torch operations; with `own` true it calls the package.

Sizes: the GPT-S decoder (12 heads of 64, a context of 1,024, V = 50,304) and the tied large vocabulary (100,352) of this repository's own workloads;
beside them grouped heads of 128 (32 query heads on 8), the common generic form.
"""
import importlib
import math

import torch

own = False
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _cache(kind, name, dtype, seqs, new, kv, heads, kv_heads, dim, page, layout="heads", window=0, ragged=False):
    return {"name": name, "kind": kind, "dtype": dtype, "seqs": seqs, "new": new, "kv": kv, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "layout": layout, "window": window, "ragged": ragged}


def _logits(name, dtype, rows, vocab, history, biases, mask):
    return {"name": name, "kind": "logits", "dtype": dtype, "rows": rows, "vocab": vocab, "history": history, "biases": biases, "mask": mask}


def listed():
    return [
        # a step of a small GPT-S batch: one row per sequence and layer, all latency
        _cache("append", "append_token", "bf16", 8, 1, 1000, 12, 12, 64, 16, ragged=True),
        # four long prompts arrive at once and are held in 8 bits
        _cache("append", "append_prompt_e4m3", "e4m3", 4, 2048, 2048, 32, 8, 128, 64),
        # a few short contexts are taken out of the cache again, to be kept elsewhere; pages laid out row by row
        _cache("read", "read_short", "bf16", 3, 777, 777, 12, 12, 64, 16, layout="rows", ragged=True),
        # contexts held in 8 bits come back for another pass over them
        _cache("read", "read_long_e4m3", "e4m3", 16, 4096, 4096, 32, 8, 128, 64, ragged=True),
        # one user talks to GPT-S: a token against a nearly full context
        _cache("attend", "attend_token", "bf16", 1, 1, 1000, 12, 12, 64, 16),
        # a batch of users, a token each, uneven contexts in 8 bits
        _cache("attend", "attend_tokens_e4m3", "e4m3", 64, 1, 4096, 32, 8, 128, 64, ragged=True),
        # two very long documents, a token each: the key axis is all there is to split
        _cache("attend", "attend_token_long", "bf16", 2, 1, 131072, 32, 8, 128, 64),
        # proposed tokens are checked in one pass, five per sequence
        _cache("attend", "attend_draft", "bf16", 24, 5, 2000, 32, 8, 128, 16, layout="rows", ragged=True),
        # the prompts of a GPT-S batch
        _cache("attend", "attend_prompt", "bf16", 4, 1024, 1024, 12, 12, 64, 16),
        # a chunk of a long document over what came before it
        _cache("attend", "attend_chunk", "bf16", 1, 4096, 16384, 32, 8, 128, 64),
        # GPT-S picks a token for four users: history, a few biases, a grammar
        _logits("logits_token", "f32", 4, 50304, 300, 16, True),
        # a large batch over a large vocabulary, long histories
        _logits("logits_batch", "bf16", 192, 100352, 2000, 40, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "attend", "logits", "logits"])
    if kind == "logits":
        vocab, history = _log(rng, 300, 150000), rng.choice([0, _log(rng, 1, 3000), _log(rng, 1, 3000)])
        biases = rng.choice([0, rng.randint(1, 60)])
        c = _logits("", rng.choice(["f32", "bf16"]), _log(rng, 1, max(1, min(256, 19000000 // vocab))), vocab, history, biases,
                    rng.random() < 0.6 or not (history or biases))
        del c["name"]
        return c
    dtype, dim, layout, page = rng.choice(["bf16", "e4m3"]), rng.choice([64, 128]), rng.choice(["heads", "rows"]), rng.choice([1, 8, 16, 24, 33, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8] if kv_heads <= 4 else [1, 1, 2, 4])
    seqs = _log(rng, 1, 64)
    row = kv_heads * dim                                       # elements of one token's keys
    if kind == "append":
        new = _log(rng, 1, max(1, 8000000 // (row * seqs)))
        c = _cache(kind, "", dtype, seqs, new, new + rng.choice([0, 5, rng.randint(0, 1000)]), heads, kv_heads, dim, page, layout, ragged=rng.random() < 0.6)
    elif kind == "read":
        kv = _log(rng, 1, max(1, min(20000, 30000000 // (row * seqs))))
        c = _cache(kind, "", dtype, seqs, kv, kv, heads, kv_heads, dim, page, layout, ragged=rng.random() < 0.6)
    else:
        form = rng.choice(["token", "token", "few", "chunk", "chunk"])
        if form == "chunk":
            seqs = _log(rng, 1, 8)
            new = _log(rng, 17, 2048)
            kv = min(new + rng.choice([0, _log(rng, 1, 8000)]), max(new, 1000000000 // (seqs * heads * new)))
        else:
            new = 1 if form == "token" else rng.randint(2, 16)
            kv = max(new, min(_log(rng, 1, 60000), 200000000 // (row * seqs)))
        c = _cache(kind, "", dtype, seqs, new, kv, heads, kv_heads, dim, page, layout, window=rng.choice([0, 0, 0, _log(rng, 1, 3000)]), ragged=rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """(new tokens, context with them) of each sequence: all alike, or uneven ones that depend on nothing but the case."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * n, [case["kv"]] * n
    part = [0.25 + 0.75 * ((0.381966 + i * 0.618034) % 1.0) for i in range(n)]
    kv = [max(1, round(case["kv"] * p)) for p in part]
    if case["kind"] == "read":
        return kv, kv
    return [max(1, min(k, round(case["new"] * (part[-1 - i] if case["new"] > 16 else 1)))) for i, k in enumerate(kv)], kv


def _power(b):
    """2^(b - 127) in 32 bits, for scale bytes b"""
    return (b.int() << 23).view(torch.float32).unsqueeze(-1)


def _held(x, scale):
    """What e4m3 numbers and their scale bytes (2^(b - 127) for every row) stand for."""
    return x.float() * _power(scale)


def _quantise(x):
    """Rows of the last axis as e4m3 numbers with one scale byte b: 2^(b - 127) is the smallest power of two by which the row's largest value fits 448, between
    2^-100 and 2^7."""
    x = x.float()
    mant, power = torch.frexp(x.abs().amax(-1))               # amax = mant * 2^power, mant in [0.5, 1); 448 = 0.875 * 2^9
    b = torch.where(mant > 0, power - 9 + (mant > 0.875), -100).clamp(-100, 7) + 127
    return (x / _power(b)).clamp(-448.0, 448.0).to(E4M3), b.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    if case["kind"] == "logits":
        return _prepare_logits(case, g, rand)
    new, kv = _lengths(case)
    hk, d, page, rows = case["kv_heads"], case["dim"], case["page"], sum(new)
    per = [-(-k // page) for k in kv]
    n_pages = sum(per) + 3
    # the pages of a cache that has been in use lie anywhere, and what a sequence does not use of its row of the table is -1
    at, column = torch.tensor([sum(per[:i]) for i in range(len(per))], device=DEV)[:, None], torch.arange(max(per), device=DEV)
    free = torch.randperm(n_pages, generator=g, device=DEV)
    table = torch.where(column < torch.tensor(per, device=DEV)[:, None], free[(at + column).clamp_(max=n_pages - 1)], -1).int()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = {"case": case, "starts": i32(starts), "kv": i32(kv), "pages": table, "max_new": max(new), "max_kv": max(kv), "rows": rows, "scales": None, "handle": None}
    # queries, keys and values of the new tokens are views of one projection's output
    qkv = rand(rows, (case["heads"] + 2 * hk) * d).bfloat16()
    s["q"], s["k"], s["v"] = (t.view(rows, -1, d) for t in qkv.split([case["heads"] * d, hk * d, hk * d], 1))
    shape = (n_pages, hk, page, d) if case["layout"] == "heads" else (n_pages, page, hk, d)
    # values grow and shrink from head to head, as a model's do
    size = torch.exp2(torch.arange(hk, device=DEV) % 5 - 2.0).view((1, hk, 1, 1) if case["layout"] == "heads" else (1, 1, hk, 1))
    pools, scales = [], []
    for _ in range(2):
        x = rand(*shape).bfloat16().mul_(size)
        if case["dtype"] == "e4m3":
            x, b = _quantise(x)
            scales.append(b if case["layout"] == "heads" else b.transpose(1, 2).contiguous())
        pools.append(x if case["layout"] == "heads" else x.transpose(1, 2))
    s["pool"], s["scales"] = pools, scales or None
    return s


def _prepare_logits(case, g, rand):
    rows, vocab, n = case["rows"], case["vocab"], case["history"]
    rnd = lambda hi, *s: torch.randint(0, hi, s, generator=g, device=DEV, dtype=torch.int32)  # noqa: E731
    s = {"case": case, "logits": (rand(rows, vocab) * 3).to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16), "history": None, "penalties": None, "bias": None, "mask": None}
    if n:
        # text repeats itself: a few tokens make up most of it
        common = (vocab * torch.rand(rows, n, generator=g, device=DEV) ** 4).int().clamp_(max=vocab - 1)
        length = (torch.arange(rows, device=DEV) * 7 % (n + 1)).int()
        length[0] = n
        s["history"] = {"tokens": common, "n_tokens": length, "n_prompt": (length.float() * 0.4).int()}
        s["penalties"] = {"repetition": 1.0 + 0.5 * torch.rand(rows, generator=g, device=DEV), "presence": 0.4 * torch.rand(rows, generator=g, device=DEV),
                          "frequency": 0.3 * torch.rand(rows, generator=g, device=DEV)}
    if case["biases"]:
        s["bias"] = {"bias_ids": rnd(vocab, rows, case["biases"]), "bias": rand(rows, case["biases"]) * 2}
    if case["mask"]:
        words = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g, device=DEV)
        s["mask"] = words.to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _own(state) if own else {"append": _append, "read": _read, "attend": _attend, "logits": _process}[state["case"]["kind"]](state)


def _own(s):
    serving = importlib.import_module("open-flapping-airplanes_b200").serving
    c = s["case"]
    if c["kind"] == "logits":
        return serving.logits_process(s["logits"], **(s["history"] or {}), **(s["penalties"] or {}), **(s["bias"] or {}), mask=s["mask"])
    if s["handle"] is None:                                    # a program makes these once and keeps them
        s["handle"] = (serving.KVCache(*s["pool"], *(s["scales"] or ())), serving.KVBatch(s["starts"], s["kv"], s["pages"], max_new=s["max_new"], max_kv=s["max_kv"]))
    cache, batch = s["handle"]
    if c["kind"] == "append":
        serving.kv_append(cache, batch, s["k"], s["v"])
        return s["pool"], s["scales"]
    if c["kind"] == "read":
        return serving.kv_read(cache, batch, s["rows"])
    return serving.paged_attention(cache, batch, s["q"], window=c["window"], with_lse=True)


def _places(s):
    """Sequence, index in its chunk, position, page and row in the page of every new row."""
    page = s["case"]["page"]
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.bucketize(row, s["starts"].long(), right=True) - 1
    t = row - s["starts"].long()[seq]
    pos = (s["kv"] - s["starts"].diff()).long()[seq] + t
    return seq, t, pos, s["pages"].long()[seq, pos // page], pos % page


def _append(s):
    _, _, _, page, at = _places(s)
    new, scales = (s["k"], s["v"]), s["scales"]
    if scales:
        (new_k, b_k), (new_v, b_v) = _quantise(s["k"]), _quantise(s["v"])
        new = (new_k, new_v)
        scales[0][page, :, at] = b_k
        scales[1][page, :, at] = b_v
    s["pool"][0].view(_bits(s))[page, :, at] = new[0].view(_bits(s))
    s["pool"][1].view(_bits(s))[page, :, at] = new[1].view(_bits(s))
    return s["pool"], s["scales"]


def _bits(s):
    """Whole numbers of the stored type's size: what torch can scatter in every version."""
    return torch.uint8 if s["scales"] else torch.int16


def _rows(s, which, page, at):
    """Cached rows, in 32 bits."""
    x = s["pool"][which].view(_bits(s))[page, :, at].view(s["pool"][which].dtype)
    return _held(x, s["scales"][which][page, :, at]) if s["scales"] else x.float()


def _read(s):
    _, _, _, page, at = _places(s)
    return _rows(s, 0, page, at).bfloat16(), _rows(s, 1, page, at).bfloat16()


def _attend(s):
    c = s["case"]
    d, hk = c["dim"], c["kv_heads"]
    group = c["heads"] // hk
    n, most, new = c["seqs"], s["max_kv"], s["max_new"]
    key = torch.arange(most, device=DEV)
    page = s["pages"].long().clamp(min=0)[:, key // c["page"]]                                   # [n, most]
    at = (key % c["page"]).expand(n, -1)
    k, v = (_rows(s, w, page, at).transpose(1, 2) for w in (0, 1))                               # [n, hk, most, d]
    row = (s["starts"].long()[:-1, None] + torch.arange(new, device=DEV)).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().view(n, new, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * new, d)
    pos = (s["kv"] - s["starts"].diff()).long()[:, None] + torch.arange(new, device=DEV)         # [n, new]
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    seen = seen[:, None, None].expand(n, 1, group, new, most).reshape(n, 1, group * new, most)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v).div_(total).view(n, hk, group, new, d)
    lse = (top + total.log()).view(n, hk, group, new)
    seq, t, _, _, _ = _places(s)
    return o[seq, :, :, t].reshape(s["rows"], c["heads"], d).bfloat16(), lse[seq, :, :, t].reshape(s["rows"], c["heads"])


def _process(s):
    c = s["case"]
    x = s["logits"].float()
    if s["penalties"]:
        h, p = s["history"], s["penalties"]
        i = torch.arange(c["history"], device=DEV)
        here = i < h["n_tokens"][:, None]
        made = (here & (i >= h["n_prompt"][:, None])).float()
        tokens = h["tokens"].long()
        seen = torch.zeros_like(x).scatter_add_(1, tokens, here.float()) > 0
        count = torch.zeros_like(x).scatter_add_(1, tokens, made)
        r = p["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - p["frequency"][:, None] * count - p["presence"][:, None] * (count > 0)
    if s["bias"]:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias"]["bias_ids"].long(), s["bias"]["bias"])
    if c["mask"]:
        at = torch.arange(c["vocab"], device=DEV)
        x = x.masked_fill((s["mask"][:, at // 32] >> (at % 32)) & 1 == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------ work, and the values in 64 bits
def work(case):
    if case["kind"] == "logits":
        n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * n * size + (n / 8 if case["mask"] else 0) + case["rows"] * (4 * case["history"] + 8 * case["biases"]), "flops": 4 * n}
    new, kv = _lengths(case)
    hk, h, d = case["kv_heads"], case["heads"], case["dim"]
    held = d + 1 if case["dtype"] == "e4m3" else 2 * d         # bytes of one cached row
    if case["kind"] in ("append", "read"):
        return {"bytes": sum(new) * hk * 2 * (2 * d + held), "flops": sum(new) * hk * d}
    reach, pairs = 0, 0
    for n, k in zip(new, kv):
        w = min(case["window"] or k, k)
        reach += min(k, n - 1 + w)                             # keys that some row sees
        first = min(k - n + 1, w)                              # of the first row; each further row sees one more, up to w
        grow = min(n - 1, w - first)
        pairs += n * first + grow * (grow + 1) // 2 + (n - 1 - grow) * grow
    return {"bytes": reach * hk * 2 * held + sum(new) * h * (4 * d + 4), "flops": 4 * d * h * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(s)
    new, kv = _lengths(case)
    page, d, hk, group = case["page"], case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    table, bits = s["pages"].tolist(), _bits(s)

    def context(which, i, first, last):
        """Cached rows [first, last) of sequence i in 64 bits, [head, row, d]"""
        pages = torch.tensor(table[i][first // page:-(-last // page)], device=DEV)
        x = s["pool"][which].view(bits)[pages].view(s["pool"][which].dtype).double()                # [pages, hk, page, d]
        if s["scales"]:
            x = x * 2.0 ** (s["scales"][which][pages].double() - 127)[..., None]
        skip = first - first // page * page
        return x.transpose(0, 1).reshape(hk, -1, d)[:, skip:skip + last - first]

    if case["kind"] == "read":
        return tuple(torch.cat([context(w, i, 0, k) for i, k in enumerate(kv)], 1).transpose(0, 1) for w in (0, 1))
    if case["kind"] == "append":
        pools = [p.double() for p in s["pool"]]
        at = 0
        for i, (n, k) in enumerate(zip(new, kv)):
            where = torch.arange(k - n, k, device=DEV)
            pages = s["pages"][i].long()[where // page]
            for w, x in enumerate((s["k"][at:at + n].double(), s["v"][at:at + n].double())):
                if s["scales"]:
                    x = x.cpu()                                # its powers of two and logarithms of them are exact
                    e = torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(-100, 7)
                    s["scales"][w][pages, :, where % page] = (e + 127).to(torch.uint8).to(DEV)
                    u = x / 2.0 ** e[..., None]
                    # the numbers of e4m3 are 2^-9 apart below 2^-6, and an eighth of their power of two above it; halves go to the even one
                    step = 2.0 ** (torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
                    x = (torch.round(u / step) * step).clamp(-448, 448).to(DEV)
                pools[w][pages, :, where % page] = x
            at += n
        return pools, s["scales"]
    outs, sums, at = [], [], 0
    for i, (n, k) in enumerate(zip(new, kv)):
        first = max(0, k - n + 1 - case["window"]) if case["window"] else 0
        keys, values = context(0, i, first, k), context(1, i, first, k)
        pos, key = torch.arange(k - n, k, device=DEV)[:, None], torch.arange(first, k, device=DEV)
        hidden = (key > pos) | (key <= pos - case["window"] if case["window"] else key < 0)
        o, z = [], []
        for h in range(case["heads"]):
            x = (s["q"][at:at + n, h].double() @ keys[h // group].T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            z.append(torch.logsumexp(x, 1))
            o.append(torch.exp(x - z[-1][:, None]) @ values[h // group])
        outs.append(torch.stack(o, 1))
        sums.append(torch.stack(z, 1))
        at += n
    return torch.cat(outs), torch.cat(sums)


def _exact_logits(s):
    c = s["case"]
    x = s["logits"].double()
    for b in range(c["rows"]):
        if s["penalties"]:
            n, first = int(s["history"]["n_tokens"][b]), int(s["history"]["n_prompt"][b])
            text = s["history"]["tokens"][b, :n].long()
            r, f, p = (float(s["penalties"][k][b]) for k in ("repetition", "frequency", "presence"))
            seen = torch.unique(text)
            x[b, seen] = torch.where(x[b, seen] > 0, x[b, seen] / r, x[b, seen] * r)
            made = torch.bincount(text[first:], minlength=c["vocab"])
            x[b] -= f * made + p * made.clamp(max=1)
        if s["bias"]:
            x[b].index_add_(0, s["bias"]["bias_ids"][b].long(), s["bias"]["bias"][b].double())
    if c["mask"]:
        words = s["mask"].long() & 0xFFFFFFFF
        allowed = torch.stack([(words >> i) % 2 for i in range(32)], -1).flatten(1)[:, :c["vocab"]] == 1
        x[~allowed] = -math.inf
    return x
