"""The serving operators over the 8-bit KV cache and the token log probabilities: cases, inputs, plain forms.

Cases of three kinds (`op`):

  append    rows of keys and values into the pages of an 8-bit cache, then the values that the touched pages stand for
  attend    attention of query rows over an 8-bit cache, causal, with an optional sliding window and first tokens (sinks)
  logprobs  log probabilities of given tokens, entropy and top alternatives of rows of logits

The cache is paged: 16 tokens a page, int8 values, one f32 scale per (page, layer, kv head) for the keys and one for the
values; keys [page][layer][kv_head][16][dim], values [page][layer][kv_head][dim][16].
"""
import math
import os
import sys

import torch

own = False

PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one generated token enters the cache of one sequence: the smallest call, between the QKV product and the attention
        dict(name="append_step", op="append", seqs=1, rows=1, ragged=False, past=512, heads=8, dim=128, layers=2, type="f32"),
        # eight prompts of up to 4096 tokens enter their caches (long-context batch), in the f32 of the layer stack
        dict(name="append_prompts", op="append", seqs=8, rows=4096, ragged=True, past=37, heads=8, dim=128, layers=1, type="f32"),
        # a single decode step over 512 cached positions: 32 query / 8 kv heads
        dict(name="step_512", op="attend", seqs=1, rows=1, ragged=False, past=512, q_heads=32, heads=8, dim=128, layers=2, type="f32", window=0, sinks=0),
        # eight long utterances (4096-token prompt and 2000 frames) decoded together
        dict(name="steps_8_long", op="attend", seqs=8, rows=1, ragged=True, past=6095, q_heads=32, heads=8, dim=128, layers=1, type="f32", window=0, sinks=0),
        # a full continuous batch: 64 utterances of up to 1024 prompt tokens and 1500 frames
        dict(name="steps_64", op="attend", seqs=64, rows=1, ragged=True, past=2523, q_heads=32, heads=8, dim=128, layers=1, type="bf16", window=0, sinks=0),
        # one sequence at the end of the longest context the model takes
        dict(name="step_32k", op="attend", seqs=1, rows=1, ragged=False, past=32767, q_heads=32, heads=8, dim=128, layers=1, type="f16", window=0, sinks=0),
        # endless streams with a bounded view: three drafted tokens each, a window and four first tokens
        dict(name="steps_window", op="attend", seqs=16, rows=3, ragged=True, past=30001, q_heads=16, heads=4, dim=64, layers=1, type="bf16", window=4000, sinks=4),
        # the 1024-token prompt of a cloned voice, in the f32 of the layer stack
        dict(name="prompt_1024", op="attend", seqs=1, rows=1024, ragged=False, past=0, q_heads=32, heads=8, dim=128, layers=1, type="f32", window=0, sinks=0),
        # two long prompts
        dict(name="prompts_4096", op="attend", seqs=2, rows=4096, ragged=True, past=0, q_heads=32, heads=8, dim=128, layers=1, type="bf16", window=0, sinks=0),
        # a long prompt under a sliding window, behind a cached prefix, in a narrow head
        dict(name="prompt_window", op="attend", seqs=1, rows=8191, ragged=False, past=333, q_heads=16, heads=4, dim=64, layers=1, type="f16", window=1000, sinks=16),
        # the next token's distribution with the tokens outside the semantic range masked, as the frame loop samples it
        dict(name="logprobs_step", op="logprobs", rows=1, vocab=155648, top=20, masked=True, type="f32"),
        # a whole prompt scored: every position's next token
        dict(name="logprobs_prompt", op="logprobs", rows=512, vocab=155648, top=8, masked=False, type="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "steps", "steps", "prompt", "prompt", "logprobs"])
    kv = rng.choice(["f32", "f16", "bf16"])
    dim, heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8])
    if kind == "append":
        seqs = _log(rng, 1, 16)
        rows = _log(rng, 1, min(4096, 32768 // seqs))
        return dict(op="append", seqs=seqs, rows=rows, ragged=rng.random() < 0.5, past=rng.choice([0, rng.randrange(4000)]), heads=heads, dim=dim, layers=rng.choice([1, 2]), type=kv)
    if kind == "logprobs":
        rows = _log(rng, 1, 512)
        return dict(op="logprobs", rows=rows, vocab=_log(rng, 1000, 155648), top=rng.choice([0, 1, 5, 20, 32]), masked=rng.random() < 0.3, type=kv)
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    if kind == "steps":
        seqs = _log(rng, 1, 64)
        past, rows = _log(rng, 1, min(32000, 160000 // seqs)), rng.choice([1, 1, 1, 2, 3, 5, 9])
    else:
        seqs = _log(rng, 1, 4)
        rows = _log(rng, 17, 4096 // seqs)
        past = rng.choice([0, rng.randrange(2000)])
        group = min(group, 32 // heads)
    window = rng.choice([0, 0, _log(rng, 1, max(2, past + rows))])
    sinks = rng.choice([0, 1, 4, 30]) if window else 0
    return dict(op="attend", seqs=seqs, rows=rows, ragged=rng.random() < 0.6, past=past, q_heads=heads * group, heads=heads, dim=dim, layers=1, type=kv, window=window, sinks=sinks)


def _lengths(case):
    """Rows and cached positions of each sequence: by the case alone."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["rows"]] * n, [case["past"]] * n
    part = [((b * 37 + n - 1) % n + 1) / n for b in range(n)]
    rows = [max(1, round(case["rows"] * (0.3 + 0.7 * part[b]))) for b in range(n)]
    past = [round(case["past"] * (0.1 + 0.9 * part[n - 1 - b])) for b in range(n)]
    return rows, past


def _visible(case):
    """(query row, key) pairs that the masks leave, keys that some row of their sequence sees."""
    rows, past = _lengths(case)
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for t, p0 in zip(rows, past):
        if not w:
            pairs += t * p0 + t * (t + 1) // 2
            keys += p0 + t
            continue
        for p in range(p0, p0 + t):
            lo = max(0, p + 1 - w)
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, p0 + 1 - w)
        keys += p0 + t - lo + min(s, lo)
    return pairs, keys


def work(case):
    e = ITEM[case["type"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * e + case["rows"] * (12 + 8 * case["top"]), flops=6 * n)
    rows, past = _lengths(case)
    hd = case["heads"] * case["dim"]
    if case["op"] == "append":
        held = sum(t + p % PAGE for t, p in zip(rows, past))  # rows of the touched pages: what is read back
        return dict(bytes=2 * hd * (sum(rows) * (e + 1) + held * (1 + 4)), flops=2 * hd * (4 * sum(rows) + held))
    pairs, keys = _visible(case)
    q = sum(rows) * case["q_heads"] * case["dim"]
    scales = 8 * case["heads"] * keys / PAGE
    return dict(bytes=2 * q * e + 2 * keys * hd + scales, flops=4 * case["dim"] * case["q_heads"] * pairs)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(case, g, rows, past):
    """A cache that holds `past` positions of each sequence (normal values, page scales that differ), with room for `rows`
    more, in pages in no order; and the table of each sequence's pages."""
    need = [(p + t + PAGE - 1) // PAGE for t, p in zip(rows, past)]
    total, ld = sum(need), max(need)
    shape = (total + 3, case["layers"], case["heads"])
    order = torch.randperm(total + 3, generator=g, device="cuda").int()
    at = torch.tensor([0] + need[:-1]).cumsum(0).cuda()
    col = torch.arange(ld, device="cuda")
    table = order[(at[:, None] + col).clamp_(max=total + 2)].contiguous()
    values = []
    for tail in ((PAGE, case["dim"]), (case["dim"], PAGE)):
        x = torch.empty(shape + tail, dtype=torch.int8, device="cuda")
        step = max(1, (1 << 26) // max(1, x[0].numel()))
        for i in range(0, shape[0], step):
            n = x[i : i + step].shape
            x[i : i + step] = torch.randn(n, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        values += [x, torch.rand(shape, generator=g, device="cuda").mul_(0.02).add_(0.02)]
    return dict(k=values[0], k_scale=values[1], v=values[2], v_scale=values[3], table=table)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    if case["op"] == "logprobs":
        rows, n = case["rows"], case["vocab"]
        x = torch.randn((rows, n), generator=g, device="cuda").mul_(3.0)
        if case["masked"]:
            x[:, : n - max(32, n // 38)] = -math.inf
        targets = torch.randint(n - max(32, n // 38) if case["masked"] else 0, n, (rows,), generator=g, device="cuda").int()
        return dict(case=case, logits=x.to(t), targets=targets)
    rows, past = _lengths(case)
    total = sum(rows)
    s = dict(case=case, past=_ints(past), row_start=_ints([sum(rows[:b]) for b in range(len(rows) + 1)]), **_pages(case, g, rows, past))

    def normal(heads, std):
        return torch.randn((total, heads, case["dim"]), generator=g, device="cuda").mul_(std).to(t)

    if case["op"] == "append":
        s.update(new_k=normal(case["heads"], 1.3), new_v=normal(case["heads"], 0.9))
        back = [p % PAGE for p in past]
        s.update(back_past=_ints([p - b for p, b in zip(past, back)]))
        s.update(back_start=_ints([sum(rows[:b]) + sum(back[:b]) for b in range(len(rows) + 1)]))
        s.update(back_rows=total + sum(back), back_max=max(r + b for r, b in zip(rows, back)))
    else:
        s.update(q=normal(case["q_heads"], 1.5))
    return s


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[s["case"]["op"]](s)


# ---- the framework's operators ----


def _own(s):
    at = os.path.join(os.getcwd(), "s2.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import s2k

    case = s["case"]
    if case["op"] == "logprobs":
        return list(s2k.logprobs(s["logits"], s["targets"], n_top=case["top"]))[: 4 if case["top"] else 2]
    cache = s2k.KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    layer = case["layers"] - 1
    if case["op"] == "append":
        cache.append(layer, s["new_k"], s["new_v"], s["past"], s["table"], row_start=s["row_start"], max_rows=case["rows"])
        return list(cache.read(layer, s["back_rows"], s["back_past"], s["table"], row_start=s["back_start"], max_rows=s["back_max"]))
    return [cache.attend(layer, s["q"], s["past"], s["table"], row_start=s["row_start"], max_rows=case["rows"], window=case["window"], sinks=case["sinks"])]


# ---- plain forms ----


def _flat(past, row_start, n):
    """Sequence and position of each of n rows."""
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(row_start, row, right=True) - 1
    return seq, past[seq].long() + row - row_start[seq]


def _append(s):
    case = s["case"]
    layer, hd, pool = case["layers"] - 1, case["heads"] * case["dim"], s["k"].shape[0]
    seq, pos = _flat(s["past"], s["row_start"], s["new_k"].shape[0])
    page, slot = s["table"][seq, pos // PAGE].long(), pos % PAGE
    kept = s["past"] % PAGE  # slots of each sequence's page of `past` that hold older tokens
    first = s["table"][torch.arange(case["seqs"], device="cuda"), s["past"].long() // PAGE].long()
    older = torch.zeros(pool, dtype=torch.int32, device="cuda").index_put_((first,), kept)
    out = []
    for name, x in (("k", s["new_k"]), ("v", s["new_v"])):
        held, scales = s[name][:, layer], s[name + "_scale"][:, layer]
        held = held if name == "k" else held.transpose(2, 3)  # [page][head][slot][dim]
        x = x.float()
        amax = torch.zeros((pool, case["heads"]), device="cuda").scatter_reduce_(0, page[:, None].expand(-1, case["heads"]), x.abs().amax(2), "amax")
        was = scales * (older > 0)[:, None]
        now = torch.maximum(was, amax / torch.full_like(amax, 127.0))  # a quotient by a number is a product with its reciprocal
        # older tokens of the page, under the scale it has now; quotients in 64 bits, for values next to a half
        values = held[first].double() * scales[first].double()[:, :, None, None]
        again = (values / now[first].double()[:, :, None, None]).nan_to_num_(0.0).round_().clamp_(-127, 127)
        mask = (torch.arange(PAGE, device="cuda") < kept[:, None])[:, None, :, None]
        held[first] = torch.where(mask, again.to(torch.int8), held[first])
        new = (x.double() / now[page].double()[:, :, None]).nan_to_num_(0.0).round_().clamp_(-127, 127)
        held[page, :, slot] = new.to(torch.int8)
        touched = torch.zeros(pool, dtype=torch.bool, device="cuda").index_fill_(0, page, True)
        scales.copy_(torch.where(touched[:, None], now, scales))
        seq_b, pos_b = _flat(s["back_past"], s["back_start"], s["back_rows"])
        page_b = s["table"][seq_b, pos_b // PAGE].long()
        out.append(held[page_b, :, pos_b % PAGE].float() * scales[page_b][:, :, None])
    return out


def _attend(s):
    case, q = s["case"], s["q"]
    layer, B, T, Hk, hd = case["layers"] - 1, case["seqs"], case["rows"], case["heads"], case["dim"]
    G = case["q_heads"] // Hk
    n = s["table"].shape[1]
    pages = s["table"].long()
    k = (s["k"][:, layer][pages].float() * s["k_scale"][:, layer][pages][..., None, None]).transpose(1, 2).reshape(B, Hk, n * PAGE, hd)
    v = (s["v"][:, layer][pages].float() * s["v_scale"][:, layer][pages][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, Hk, n * PAGE, hd)
    seq, pos = _flat(s["past"], s["row_start"], q.shape[0])
    at = pos - s["past"][seq]
    padded = torch.zeros((B, T, Hk, G, hd), device="cuda")
    padded[seq, at] = q.float().view(-1, Hk, G, hd)
    x = padded.permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, hd)
    p = (s["past"][:, None] + torch.arange(T, device="cuda"))[:, None, None, :, None]
    j = torch.arange(n * PAGE, device="cuda")
    hidden = j > p
    if case["window"]:
        hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
    a = (x @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(B, Hk, G, T, n * PAGE).masked_fill_(hidden, -math.inf)
    a = a.sub_(a.amax(-1, keepdim=True)).exp_()
    total = a.sum(-1, keepdim=True)
    o = (a.view(B, Hk, G * T, n * PAGE) @ v).view(B, Hk, G, T, hd).div_(total)
    return [o.permute(0, 3, 1, 2, 4)[seq, at].reshape(q.shape).to(q.dtype)]


def _logprobs(s):
    x, k = s["logits"].float(), s["case"]["top"]
    rows, n = x.shape
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    peak = d == 0  # the largest values add one each: kept apart, so that a sure row's small rest is not lost beside them
    count = peak.sum(1, dtype=torch.float32)
    rest = torch.where(peak, torch.zeros_like(e), e).sum(1)
    log_total = count.log() + (rest / count).log1p()
    entropy = log_total - torch.where(e > 0, d * e, torch.zeros_like(e)).sum(1) / (count + rest)
    out = [d.gather(1, s["targets"].long()[:, None])[:, 0] - log_total, entropy]
    if k:
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
        ids = (order + (n - 1 - torch.arange(n, device="cuda"))).topk(k, 1).indices  # ties: the lowest index
        out += [ids.int(), d.gather(1, ids) - log_total[:, None]]
    return out


# ---- from the definitions, in 64 bits ----


def _exact_append(s):
    case = s["case"]
    layer, rows, past = case["layers"] - 1, *_lengths(case)
    table, out, start = s["table"].tolist(), [], [0]
    for t in rows:
        start.append(start[-1] + t)
    for name, new in (("k", s["new_k"]), ("v", s["new_v"])):
        got = []
        for b, (t, p0) in enumerate(zip(rows, past)):
            keep = p0 % PAGE
            x = new[start[b] : start[b + 1]].double()
            before = torch.zeros((0,) + tuple(x.shape[1:]), dtype=torch.float64, device="cuda")
            first_scale = torch.zeros(x.shape[1], dtype=torch.float64, device="cuda")
            if keep:
                page = table[b][p0 // PAGE]
                ints = s[name][page, layer].double()
                ints = ints.permute(1, 0, 2) if name == "k" else ints.permute(2, 0, 1)
                first_scale = s[name + "_scale"][page, layer].double()
                before = (ints * first_scale[None, :, None])[:keep]
            both = torch.cat([before, x])
            pad = -len(both) % PAGE
            groups = torch.nn.functional.pad(both, (0, 0, 0, 0, 0, pad)).view(-1, PAGE, *both.shape[1:])
            fresh = torch.cat([torch.zeros_like(before), x])
            top = torch.nn.functional.pad(fresh, (0, 0, 0, 0, 0, pad)).view(groups.shape).abs().amax((1, 3))
            scale = (top / 127).float().double()  # a scale is held in 32 bits
            scale[0] = torch.maximum(scale[0], first_scale)
            unit = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None, :, None]
            got.append(((groups / unit).round() * scale[:, None, :, None]).view(-1, *both.shape[1:])[: len(both)])
        out.append(torch.cat(got))
    return out


def _exact_attend(s):
    case = s["case"]
    rows, past = _lengths(case)
    layer, hd, G = case["layers"] - 1, case["dim"], case["q_heads"] // case["heads"]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (t, p0) in enumerate(zip(rows, past)):
        used = s["table"][b, : (p0 + t + PAGE - 1) // PAGE].long()
        for h in range(case["heads"]):
            k = s["k"][used, layer, h].double() * s["k_scale"][used, layer, h].double()[:, None, None]
            v = s["v"][used, layer, h].double() * s["v_scale"][used, layer, h].double()[:, None, None]
            k, v = k.reshape(-1, hd)[: p0 + t], v.permute(0, 2, 1).reshape(-1, hd)[: p0 + t]
            j = torch.arange(p0 + t, device="cuda")
            for lo in range(0, t, 2048):
                hi = min(t, lo + 2048)
                q = s["q"][at + lo : at + hi, h * G : (h + 1) * G].double()
                p = torch.arange(p0 + lo, p0 + hi, device="cuda")[:, None]
                seen = j <= p
                if case["window"]:
                    seen = seen & ((j > p - case["window"]) | (j < case["sinks"]))
                score = torch.einsum("tgd,jd->gtj", q, k) / math.sqrt(hd)
                w = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), -1)
                out[at + lo : at + hi, h * G : (h + 1) * G] = torch.einsum("gtj,jd->tgd", w, v)
        at += t
    return [out]


def _exact_logprobs(s):
    logp, entropy, top = [], [], []
    for x, target in zip(s["logits"], s["targets"].tolist()):
        z = torch.log_softmax(x.double(), 0)
        logp.append(z[target])
        entropy.append(-torch.where(z > -math.inf, z.exp() * z, torch.zeros_like(z)).sum())
        top.append(torch.topk(z, s["case"]["top"]).values if s["case"]["top"] else z[:0])
    out = [torch.stack(logp), torch.stack(entropy)]
    return out + [None, torch.stack(top)] if s["case"]["top"] else out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](s)
