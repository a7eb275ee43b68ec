"""The operators of an 8-bit cache and of drafted tokens: what is measured of them, their plain forms and their exact values.

store    a step's queries, keys and values: queries and keys are rotated, keys and values go into the pages of the cache
         as 8-bit floats (e4m3) with one power of two for each token and head (`ops.rope_kv_q8`)
attend   attention of a step's query rows over such a cache: steps of single tokens, of a few drafted tokens, of whole
         prompts and of pieces of them (`ops.attention_q8`)
verify   a step's drafted tokens against the target model's logits, from given uniform numbers: how many are kept and
         which token follows them (`ops.verify_drafts`)

A page holds 64 tokens of every kv head, one head after the other, in 128 * (head size + 1) bytes each:

    keys     byte  (t * P + p) * 256 + i * 16 + e        of token 16 t + i, element 16 p + e   (P = head size / 16)
    values   byte  ((c * 4 + g) * 16 + i) * 16 + 4 t + r  of token 16 t + 4 g + r, element 16 c + i
    scales   of the keys: byte 4 i + t of token 16 t + i; of the values: byte 16 g + 4 t + r of token 16 t + 4 g + r

An element is its e4m3 value times 2^(scale - 127); the power is the smallest that brings the largest magnitude of the
token's head within e4m3's 448.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 64


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of eight sequences of the Llama 3.2 1B shape: a launch's latency is what counts
        {"name": "store_decode_8", "op": "store", "n_seq": 8, "q_lo": 1, "q_hi": 1, "past_lo": 2048, "past_hi": 2303, "heads": 32, "kv": 8, "hd": 64},
        # the prompts of a batch of sixteen requests with the head layout of the Llama 3.2 3B shape
        {"name": "store_prompts_ragged", "op": "store", "n_seq": 16, "q_lo": 128, "q_hi": 2048, "past_lo": 0, "past_hi": 0, "heads": 24, "kv": 8, "hd": 128},
        # one sequence decoding alone
        {"name": "attend_single_1", "op": "attend", "n_seq": 1, "q_lo": 1, "q_hi": 1, "past_lo": 2300, "past_hi": 2300, "heads": 32, "kv": 8, "hd": 64, "window": 0},
        # the benchmark's batch of 64 after 2,048-token prompts
        {"name": "attend_single_64", "op": "attend", "n_seq": 64, "q_lo": 1, "q_hi": 1, "past_lo": 2048, "past_hi": 2303, "heads": 32, "kv": 8, "hd": 64, "window": 0},
        # the Llama 3.1 8B workload: 32 requests of very unequal lengths, mid-generation
        {"name": "attend_single_ragged", "op": "attend", "n_seq": 32, "q_lo": 1, "q_hi": 1, "past_lo": 63, "past_hi": 8191, "heads": 32, "kv": 8, "hd": 128, "window": 0},
        # a few requests with very long contexts
        {"name": "attend_single_long", "op": "attend", "n_seq": 4, "q_lo": 1, "q_hi": 1, "past_lo": 20011, "past_hi": 32766, "heads": 32, "kv": 8, "hd": 64, "window": 0},
        # a step that brings up to five drafted tokens beside each sequence's own
        {"name": "attend_drafts_16", "op": "attend", "n_seq": 16, "q_lo": 1, "q_hi": 6, "past_lo": 128, "past_hi": 4089, "heads": 32, "kv": 8, "hd": 64, "window": 0},
        # one whole prompt, the benchmark's 2,048 tokens
        {"name": "attend_prompt_2048", "op": "attend", "n_seq": 1, "q_lo": 2048, "q_hi": 2048, "past_lo": 0, "past_hi": 0, "heads": 32, "kv": 8, "hd": 64, "window": 0},
        # pieces of prompts that continue sequences already in the cache
        {"name": "attend_prompts_ragged", "op": "attend", "n_seq": 8, "q_lo": 64, "q_hi": 2048, "past_lo": 0, "past_hi": 2048, "heads": 32, "kv": 8, "hd": 128, "window": 0},
        # the drafts of one sequence over Llama's vocabulary
        {"name": "verify_1", "op": "verify", "n_seq": 1, "k_lo": 4, "k_hi": 4, "vocab": 128256, "model_drafts": True},
        # eight sequences whose drafts were looked up in their own text (a draft is certain of its token)
        {"name": "verify_lookup_8", "op": "verify", "n_seq": 8, "k_lo": 0, "k_hi": 7, "vocab": 128256, "model_drafts": False},
        # a full batch with five drafts each from a draft model
        {"name": "verify_64", "op": "verify", "n_seq": 64, "k_lo": 5, "k_hi": 5, "vocab": 128256, "model_drafts": True},
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "store_prompts", "single", "single", "drafts", "prompts", "verify"])
    kv = rng.choice([1, 2, 3, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7])
    hd = rng.choice([16, 32, 48, 64, 64, 80, 128, 128, 256])
    if kind == "store":
        past = log_int(rng, 1, 8000)
        return {"op": "store", "n_seq": log_int(rng, 1, 64), "q_lo": 1, "q_hi": rng.choice([1, 1, 5]), "past_lo": past // 2, "past_hi": past, "heads": heads, "kv": kv, "hd": hd}
    if kind == "store_prompts":
        q = log_int(rng, 2, 2048)
        past = rng.choice([0, log_int(rng, 1, 4000)])
        return {"op": "store", "n_seq": log_int(rng, 1, 12), "q_lo": max(1, q // 3), "q_hi": q, "past_lo": past // 3, "past_hi": past, "heads": heads, "kv": kv, "hd": min(hd, 128)}
    window = rng.choice([0, 0, 0, log_int(rng, 1, 2000)])
    if kind == "single":
        past = log_int(rng, 1, 30000)
        n = max(1, min(log_int(rng, 1, 64), 200000 * 128 // (past * max(hd, 64))))
        return {"op": "attend", "n_seq": n, "q_lo": 1, "q_hi": 1, "past_lo": rng.randint(0, past), "past_hi": past, "heads": heads, "kv": kv, "hd": hd, "window": window}
    if kind == "drafts":
        past = log_int(rng, 1, 8000)
        return {"op": "attend", "n_seq": log_int(rng, 1, 24), "q_lo": rng.randint(1, 3), "q_hi": rng.randint(3, 9), "past_lo": rng.randint(0, past), "past_hi": past, "heads": heads, "kv": kv, "hd": min(hd, 128), "window": window}
    if kind == "prompts":
        q = log_int(rng, 17, 1700)
        past = rng.choice([0, log_int(rng, 1, 1500)])
        return {"op": "attend", "n_seq": rng.randint(1, 6), "q_lo": max(1, q // 5), "q_hi": q, "past_lo": 0, "past_hi": past, "heads": heads, "kv": kv, "hd": min(hd, 128), "window": window}
    k = rng.randint(1, 8)
    vocab = rng.choice([384, 1001, 32000, 50257, 128256])
    return {"op": "verify", "n_seq": max(1, log_int(rng, 1, 64) // (1 if k < 5 else 2)), "k_lo": rng.randint(0, k), "k_hi": k, "vocab": vocab, "model_drafts": rng.random() < 0.7}


def spread(n, lo, hi, salt):
    """n whole numbers over [lo, hi], both ends among them, in an order without pattern; the same for the same case."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(1000 * n + salt).shuffle(v)
    return v


def lengths(case):
    """Rows that each sequence brings, and the tokens it held before."""
    q = spread(case["n_seq"], case["q_lo"], case["q_hi"], 1)
    past = spread(case["n_seq"], case["past_lo"], case["past_hi"], 2)
    return q, past


# ---------------------------------------------------------------------------------------------------- the format
def quantised(x):
    """x [..., head size] float32 -> its e4m3 values (float8) and the bytes of its powers of two [...]."""
    bits = (x.view(torch.int32) & 0x7FFFFFFF).amax(-1)
    power = (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).int()       # amax <= 448 * 2^power
    power = power.clamp(-126, 127)
    vals = torch.ldexp(x, -power.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return vals, (power + 127).to(torch.uint8)


def head_bytes(hd):
    return 128 * (hd + 1)


def pages_of(k, v):
    """Keys and values [pages, kv heads, 64, head size] float32 -> pages [pages, kv heads, bytes]."""
    n, kv, _, hd = k.shape
    kq, ks = quantised(k)
    vq, vs = quantised(v)
    kb = kq.view(torch.uint8).view(n, kv, 4, 16, hd // 16, 16).permute(0, 1, 2, 4, 3, 5).reshape(n, kv, -1)
    vb = vq.view(torch.uint8).view(n, kv, 4, 4, 4, hd // 16, 16).permute(0, 1, 5, 3, 6, 2, 4).reshape(n, kv, -1)
    ks = ks.view(n, kv, 4, 16).transpose(2, 3).reshape(n, kv, -1)
    vs = vs.view(n, kv, 4, 4, 4).transpose(2, 3).reshape(n, kv, -1)
    return torch.cat([kb, vb, ks, vs], -1)


def values_of(pages, hd):
    """Pages [..., kv heads, bytes] -> keys and values [..., kv heads, 64, head size] float32."""
    lead = pages.shape[:-1]
    n = PAGE * hd
    f8 = pages[..., : 2 * n].contiguous().view(torch.float8_e4m3fn).float()
    power = pages[..., 2 * n:].float() - 127.0
    k = f8[..., :n].view(-1, 4, hd // 16, 16, 16).transpose(2, 3).reshape(-1, PAGE, hd)
    v = f8[..., n:].view(-1, hd // 16, 4, 16, 4, 4).permute(0, 4, 2, 5, 1, 3).reshape(-1, PAGE, hd)
    ks = power[..., :64].reshape(-1, 16, 4).transpose(1, 2).reshape(-1, PAGE, 1)
    vs = power[..., 64:].reshape(-1, 4, 4, 4).transpose(1, 2).reshape(-1, PAGE, 1)
    return (k * torch.exp2(ks)).view(*lead, PAGE, hd), (v * torch.exp2(vs)).view(*lead, PAGE, hd)


# ---------------------------------------------------------------------------------------------------- the inputs
def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def int32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32), device=DEV)


def prepare(case, seed):
    g = generator(seed)
    if case["op"] == "verify":
        return prepare_verify(case, g)
    n, kv, hd, heads = case["n_seq"], case["kv"], case["hd"], case["heads"]
    q_lens, past = lengths(case)
    total = sum(q_lens)
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    held = [(p + q + PAGE - 1) // PAGE for p, q in zip(past, q_lens)]       # pages of each sequence
    width = max(held) + 1
    n_slots, n_pages = n + 3, sum(held) + 2
    slots = torch.randperm(n_slots, generator=g, device=DEV)[:n].int()
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((n_slots, width), -1, dtype=torch.int32, device=DEV)
    seq_of_page = torch.as_tensor(np.repeat(np.arange(n), held), device=DEV)
    place = torch.as_tensor(np.concatenate([np.arange(h) for h in held]), device=DEV)
    table[slots.long()[seq_of_page], place] = ids[: sum(held)]
    state = {"case": case, "cu_q": int32(cu), "start_pos": int32(past), "slots": slots, "page_table": table,
             "tok_seq": int32(np.repeat(np.arange(n), q_lens)),
             "positions": int32(np.concatenate([np.arange(p, p + q) for p, q in zip(past, q_lens)])),
             "max_q_len": max(q_lens), "max_kv_len": max(p + q for p, q in zip(past, q_lens)), "page_stride": kv * head_bytes(hd)}
    # what the pages held before: the keys and values of tokens, some much larger than others
    pages = torch.empty(n_pages, kv, head_bytes(hd), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (kv * PAGE * hd))
    for a in range(0, n_pages, step):
        m = min(step, n_pages - a)
        size = torch.exp(0.5 * torch.randn(m, kv, PAGE, 1, generator=g, device=DEV))
        k = torch.randn(m, kv, PAGE, hd, generator=g, device=DEV) * size
        v = torch.randn(m, kv, PAGE, hd, generator=g, device=DEV) * size.flip(2)
        pages[a : a + m] = pages_of(k, v)
    state["cache"] = pages.view(-1)
    if case["op"] == "attend":
        state["q"] = torch.randn(total, heads * hd, generator=g, device=DEV).bfloat16()
        state["out"] = torch.empty_like(state["q"])
        scratch = {}

        def partials(count):                    # a workspace that a program keeps for its steps
            if "part" not in scratch or scratch["part"].numel() < count:
                scratch["part"] = torch.empty(count, dtype=torch.float32, device=DEV)
            return scratch["part"]
        state["scratch"] = partials
        return state
    state["qkv"] = (torch.randn(total, (heads + 2 * kv) * hd, generator=g, device=DEV)
                    * torch.exp(0.5 * torch.randn(total, 1, generator=g, device=DEV))).bfloat16()
    state["q_out"] = torch.empty(total, heads * hd, dtype=torch.bfloat16, device=DEV)
    freq = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    angle = torch.arange(state["max_kv_len"], dtype=torch.float64, device=DEV)[:, None] * freq
    state["cos"], state["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    return state


def prepare_verify(case, g):
    n, vocab = case["n_seq"], case["vocab"]
    k = spread(n, case["k_lo"], case["k_hi"], 3)
    d = sum(k)
    cu = np.concatenate([[0], np.cumsum(k)])
    temperature = torch.full((n,), 0.8, device=DEV)
    temperature[torch.arange(n, device=DEV) % 8 == 5] = 0.0                    # a greedy request among the others
    logits = 2.5 * torch.randn(d + n, vocab, generator=g, device=DEV)
    state = {"case": case, "cu_drafts": int32(cu), "temperature": temperature, "max_drafts": max(k), "logits": logits,
             "uniform": torch.rand(d + n, generator=g, device=DEV),
             "accepted": torch.empty(n, dtype=torch.int32, device=DEV), "token": torch.empty(n, dtype=torch.int32, device=DEV),
             "probs": torch.empty(d, device=DEV)}
    rows = torch.as_tensor(np.concatenate([np.arange(c, c + x) + i for i, (c, x) in enumerate(zip(cu, k))] or [[]]).astype(np.int64), device=DEV)
    if case["model_drafts"]:                    # a smaller model that agrees with the target more or less
        state["draft_logits"] = logits[rows] + 0.7 * torch.randn(d, vocab, generator=g, device=DEV)
        source = state["draft_logits"] / 0.8
    else:
        state["draft_logits"] = None
        source = logits[rows] / 0.5
    noise = -torch.log(-torch.log(torch.rand(d, vocab, generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)))
    state["draft_tokens"] = (source + noise).argmax(-1).int() if d else torch.empty(0, dtype=torch.int32, device=DEV)
    scratch = {}

    def work(count):
        if "work" not in scratch or scratch["work"].numel() < count:
            scratch["work"] = torch.empty(count, dtype=torch.uint8, device=DEV)
        return scratch["work"]
    state["scratch"] = work
    return state


# ---------------------------------------------------------------------------------------------------- a pass
def run(s):
    case = s["case"]
    if case["op"] == "store":
        if own:
            from dlgo_amd.kernels import ops
            ops.rope_kv_q8(s["qkv"], s["q_out"], case["heads"], case["kv"], case["hd"], case["hd"], False, s["cos"], s["sin"],
                           s["positions"], s["tok_seq"], s["slots"], s["page_table"], s["cache"], s["page_stride"])
        else:
            plain_store(s)
        hd = case["hd"]
        pages = s["cache"].view(-1, case["kv"], head_bytes(hd))
        # what the 8 bits stand for: e4m3 numbers, and powers of two
        return {"q": s["q_out"], "values": pages[..., : 128 * hd].view(torch.float8_e4m3fn), "scales": pages[..., 128 * hd:].view(torch.float8_e8m0fnu)}
    if case["op"] == "attend":
        if own:
            from dlgo_amd.kernels import ops
            ops.attention_q8(s["q"], s["out"], case["heads"], case["kv"], case["hd"], s["cu_q"], s["start_pos"], s["slots"], s["page_table"],
                             s["cache"], s["page_stride"], s["max_q_len"], s["max_kv_len"], window=case["window"], scratch=s["scratch"])
        else:
            plain_attend(s)
        return s["out"]
    if own:
        from dlgo_amd.kernels import ops
        ops.verify_drafts(s["logits"], s["draft_tokens"], s["cu_drafts"], s["temperature"], s["uniform"], s["accepted"], s["token"],
                          s["max_drafts"], draft_logits=s["draft_logits"], probs=s["probs"], scratch=s["scratch"])
        return {"accepted": s["accepted"], "token": s["token"], "probs": s["probs"]}
    return plain_verify(s)


# ---------------------------------------------------------------------------------------------------- plain forms
def plain_store(s):
    case = s["case"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    x = s["qkv"].float().view(-1, heads + 2 * kv, hd)
    pos = s["positions"].long()
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    a, b = x[:, : heads + kv, : hd // 2], x[:, : heads + kv, hd // 2:]
    # a product and then a product that is added without a rounding of its own (64 bits hold it): keys a last bit apart
    # would fall on either side of an 8-bit border
    turned = torch.cat([((a * cos).double() - b.double() * sin.double()).float(), ((b * cos).double() + a.double() * sin.double()).float()], -1)
    s["q_out"].copy_(turned[:, :heads].reshape(-1, heads * hd))
    kq, ks = quantised(turned[:, heads:].contiguous())
    vq, vs = quantised(x[:, heads + kv:].contiguous())
    page = s["page_table"][s["slots"][s["tok_seq"].long()].long(), pos // PAGE].long()
    place = pos % PAGE
    base = (page * kv)[:, None] + torch.arange(kv, device=DEV)
    base = base * head_bytes(hd)                                                     # of each token's head
    e = torch.arange(hd, device=DEV)
    t16, i16 = place // 16, place % 16
    at_k = ((t16 * (hd // 16))[:, None] + e // 16) * 256 + (i16 * 16)[:, None] + e % 16
    g, r = i16 // 4, i16 % 4
    at_v = ((e // 16 * 4)[None] + g[:, None]) * 256 + (e % 16 * 16)[None] + (4 * t16 + r)[:, None]
    s["cache"][base[..., None] + at_k[:, None]] = kq.view(torch.uint8)
    s["cache"][base[..., None] + PAGE * hd + at_v[:, None]] = vq.view(torch.uint8)
    s["cache"][base + 2 * PAGE * hd + (4 * i16 + t16)[:, None]] = ks
    s["cache"][base + 2 * PAGE * hd + PAGE + (16 * g + 4 * t16 + r)[:, None]] = vs


def plain_attend(s):
    case = s["case"]
    n, heads, kv, hd = case["n_seq"], case["heads"], case["kv"], case["hd"]
    group, qm = heads // kv, s["max_q_len"]
    pages = (s["max_kv_len"] + PAGE - 1) // PAGE
    pool = s["cache"].view(-1, kv, head_bytes(hd))
    table = s["page_table"][s["slots"].long()][:, :pages].long().clamp(min=0)
    k, v = values_of(pool[table], hd)                                              # [n, pages, kv, 64, hd]
    k = k.transpose(1, 2).reshape(n, kv, pages * PAGE, hd)
    v = v.transpose(1, 2).reshape(n, kv, pages * PAGE, hd)
    cu = s["cu_q"].long()
    row = cu[:-1, None] + torch.arange(qm, device=DEV)                             # [n, most rows]
    real = row < cu[1:, None]
    q = s["q"].float()[row.clamp(max=s["q"].shape[0] - 1)].view(n, qm, kv, group, hd).transpose(1, 2).reshape(n, kv, qm * group, hd)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(n, kv, qm, group, -1)
    pos = s["start_pos"].long()[:, None] + torch.arange(qm, device=DEV)
    key = torch.arange(pages * PAGE, device=DEV)
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_().view(n, kv, qm * group, -1)
    key_in = key < (s["start_pos"].long() + cu[1:] - cu[:-1])[:, None]             # tokens that the sequence holds
    v.masked_fill_(~key_in[:, None, :, None], 0.0)
    out = torch.matmul(weights, v) / weights.sum(-1, keepdim=True)
    out = out.view(n, kv, qm, group, hd).transpose(1, 2).reshape(n, qm, heads * hd)
    s["out"].copy_(out[real])


def plain_verify(s):
    n, vocab = s["temperature"].shape[0], s["logits"].shape[1]
    cu, u = s["cu_drafts"].long(), s["uniform"].double()
    d = cu[1:] - cu[:-1]
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), d + 1, output_size=s["logits"].shape[0])
    p = s["logits"].double() / t[seq, None]
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    best = s["logits"].argmax(-1)
    dseq = torch.repeat_interleave(torch.arange(n, device=DEV), d, output_size=s["draft_tokens"].shape[0])
    at = torch.arange(dseq.shape[0], device=DEV)
    row = at + dseq                                                                # the target's row for each draft
    draft = s["draft_tokens"].long()
    p_draft = p[row, draft]
    if s["draft_logits"] is None:
        q_draft = torch.ones_like(p_draft)
    else:
        q = s["draft_logits"].double() / t[dseq, None]
        q = torch.exp(q - q.amax(-1, keepdim=True))
        q /= q.sum(-1, keepdim=True)
        q_draft = q[at, draft]
    keep = torch.where(greedy[dseq], draft == best[row], u[row] * q_draft < p_draft)
    k = s["max_drafts"]
    place = cu[:-1, None] + torch.arange(k, device=DEV)
    has = torch.arange(k, device=DEV) < d[:, None]
    padded = torch.cat([keep, keep.new_zeros(1)])[torch.where(has, place, keep.shape[0])]
    accepted = padded.long().cumprod(-1).sum(-1)
    last = cu[:-1] + torch.arange(n, device=DEV) + accepted                        # the row that the next token is drawn from
    w = p[last]
    short = accepted < d                                                           # a draft was refused: what it takes away goes
    if draft.shape[0]:
        refused = (cu[:-1] + accepted).clamp(max=draft.shape[0] - 1)
        if s["draft_logits"] is None:
            less = torch.zeros_like(w)
            less[torch.arange(n, device=DEV), draft[refused]] = 1.0
        else:
            less = q[refused]
        rest = torch.where(short[:, None], (w - less).clamp(min=0), w)
        w = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    sums = w.cumsum(-1)
    target = u[cu[1:] + torch.arange(n, device=DEV)] * sums[:, -1]
    drawn = (sums <= target[:, None]).sum(-1).clamp(max=vocab - 1)
    token = torch.where(greedy, best[last], drawn)
    probs = torch.where(greedy[dseq], (draft == best[row]).double(), p_draft)
    return {"accepted": accepted.int(), "token": token.int(), "probs": probs.float()}


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "verify":
        d = sum(spread(case["n_seq"], case["k_lo"], case["k_hi"], 3))
        rows = d + case["n_seq"] + (d if case["model_drafts"] else 0)
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 12.0 * rows * case["vocab"]}
    q_lens, past = lengths(case)
    kv, hd, heads = case["kv"], case["hd"], case["heads"]
    rows = sum(q_lens)
    if case["op"] == "store":
        read = rows * (heads + 2 * kv) * hd * 2 + rows * hd * 4
        return {"bytes": float(read + rows * heads * hd * 2 + rows * kv * 2 * (hd + 1)), "flops": float(rows * (heads + kv) * hd * 3 + rows * 2 * kv * hd * 2)}
    w = case["window"]
    seen = 0                    # keys over all rows
    held = 0                    # tokens whose keys and values some row sees
    for q, p in zip(q_lens, past):
        pos = np.arange(p, p + q, dtype=np.int64)
        seen += int((np.minimum(pos + 1, w) if w else pos + 1).sum())
        held += p + q - (max(0, p - w + 1) if w else 0)
    return {"bytes": float(held * kv * 2 * (hd + 1) + 2 * rows * heads * hd * 2), "flops": 4.0 * seen * heads * hd}


# ---------------------------------------------------------------------------------------------------- exact values
def exact(case, seed):
    s = prepare(case, seed)
    return {"store": exact_store, "attend": exact_attend, "verify": exact_verify}[case["op"]](s)


def e4m3_nearest(x):
    """The e4m3 number nearest to each x (float64, magnitudes up to 448), ties to an even last place."""
    exponent = torch.frexp(x.abs().clamp(min=1e-300))[1] - 1
    step = torch.exp2((exponent.clamp(min=-6) - 3).double())
    return torch.round(x / step) * step


def exact_store(s):
    case = s["case"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    rows = s["qkv"].double().view(-1, heads + 2 * kv, hd)
    c, sn = s["cos"].double(), s["sin"].double()
    pos = s["positions"].cpu().numpy()
    on = torch.as_tensor(pos.astype(np.int64), device=DEV)
    z = torch.complex(rows[:, : heads + kv, : hd // 2], rows[:, : heads + kv, hd // 2:]) * torch.complex(c[on], sn[on])[:, None]
    turned = torch.cat([z.real, z.imag], -1)
    pages = s["cache"].view(-1, kv, head_bytes(hd))
    values = pages[..., : 128 * hd].view(torch.float8_e4m3fn).double().reshape(-1)
    table, slots, seq = s["page_table"].cpu().numpy(), s["slots"].cpu().numpy(), s["tok_seq"].cpu().numpy()
    page = torch.as_tensor(table[slots[seq], pos // PAGE].astype(np.int64), device=DEV)
    place = on % PAGE
    for what, vals in (("k", turned[:, heads:]), ("v", rows[:, heads + kv:])):
        top = vals.abs().amax(-1, keepdim=True)
        power = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=-126)
        q = e4m3_nearest(vals / torch.exp2(power))
        for e in range(hd):
            if what == "k":
                inside = (place // 16 * (hd // 16) + e // 16) * 256 + place % 16 * 16 + e % 16
            else:
                inside = PAGE * hd + (e // 16 * 4 + place % 16 // 4) * 256 + e % 16 * 16 + place // 16 * 4 + place % 4
            for h in range(kv):
                values[(page * kv + h) * 128 * hd + inside] = q[:, h, e]
    return {"q": turned[:, :heads].reshape(-1, heads * hd), "values": values.view(-1, kv, 128 * hd), "scales": None}


def exact_attend(s):
    case = s["case"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    group, w = heads // kv, case["window"]
    cu, past = s["cu_q"].cpu().tolist(), s["start_pos"].cpu().tolist()
    raw = s["cache"].view(-1, kv, head_bytes(hd))
    table = s["page_table"].cpu()[s["slots"].cpu().long()].to(DEV)
    byte_value = torch.arange(256, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn).double()
    token = torch.arange(PAGE, device=DEV)[:, None]
    e = torch.arange(hd, device=DEV)[None]
    at_k = (token // 16 * (hd // 16) + e // 16) * 256 + token % 16 * 16 + e % 16
    at_v = PAGE * hd + (e // 16 * 4 + token % 16 // 4) * 256 + e % 16 * 16 + token // 16 * 4 + token % 4
    token = token[:, 0]
    at_ks = 128 * hd + token % 16 * 4 + token // 16
    at_vs = 128 * hd + PAGE + token % 16 // 4 * 16 + token // 16 * 4 + token % 4
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for i in range(case["n_seq"]):
        length = past[i] + cu[i + 1] - cu[i]
        held = raw[table[i, : (length + PAGE - 1) // PAGE].long()]
        q = s["q"][cu[i]:cu[i + 1]].double().view(-1, kv, group, hd)
        pos = past[i] + torch.arange(q.shape[0], device=DEV)
        key = torch.arange(length, device=DEV)
        hidden = key[None] > pos[:, None]
        if w:
            hidden |= key[None] < pos[:, None] - w + 1
        for h in range(kv):
            b = held[:, h].long()
            k = (byte_value[b[:, at_k]] * torch.exp2(b[:, at_ks].double() - 127)[..., None]).reshape(-1, hd)[:length]
            v = (byte_value[b[:, at_v]] * torch.exp2(b[:, at_vs].double() - 127)[..., None]).reshape(-1, hd)[:length]
            for j in range(group):
                a = (q[:, h, j] @ k.t()) / math.sqrt(hd)
                a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
                out[cu[i]:cu[i + 1], (h * group + j) * hd:(h * group + j + 1) * hd] = a @ v
    return out


def exact_verify(s):
    cu = s["cu_drafts"].cpu().tolist()
    temperature, u, drafts = s["temperature"].cpu().tolist(), s["uniform"].cpu().tolist(), s["draft_tokens"].cpu().tolist()
    accepted, token, probs = [], [], []
    for i, temp in enumerate(temperature):
        row, k = cu[i] + i, cu[i + 1] - cu[i]
        x = s["logits"][row: row + k + 1].double().cpu()
        if temp <= 0:
            p = torch.nn.functional.one_hot(x.argmax(-1), x.shape[1]).double()
        else:
            p = torch.softmax(x / np.float64(np.float32(temp)), -1)
        if s["draft_logits"] is None or temp <= 0:
            q = torch.zeros(k, x.shape[1], dtype=torch.float64)
            q[torch.arange(k), torch.as_tensor(drafts[cu[i]:cu[i + 1]], dtype=torch.int64)] = 1.0
        else:
            q = torch.softmax(s["draft_logits"][cu[i]:cu[i + 1]].double().cpu() / np.float64(np.float32(temp)), -1)
        j = 0
        while j < k and u[row + j] * q[j, drafts[cu[i] + j]].item() < p[j, drafts[cu[i] + j]].item():
            j += 1
        rest = torch.clamp(p[j] - q[j], min=0) if j < k else p[j]
        if not rest.sum().item() > 0:
            rest = p[j]
        c = torch.cumsum(rest, 0)
        token.append(min(int(torch.searchsorted(c, u[row + k] * c[-1].item(), right=True)), x.shape[1] - 1))
        accepted.append(j)
        probs += [p[m, drafts[cu[i] + m]].item() for m in range(k)]
    return {"accepted": torch.as_tensor(accepted, dtype=torch.int32, device=DEV), "token": torch.as_tensor(token, dtype=torch.int32, device=DEV),
            "probs": torch.as_tensor(probs, dtype=torch.float64, device=DEV)}
