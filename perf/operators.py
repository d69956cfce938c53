"""Operators of a batched serving step, as measured: their inputs, their plain forms, and the calls that a user makes.

``attention``   :func:`jetspec_b200.ops.shared_prefix_attention`: a batch whose sequences share a long prefix (a system prompt, a
                document, samples of one request) in the paged pool; single decoded tokens, token trees, portions of prompts.
``verify``      :func:`jetspec_b200.ops.verify_chains`: drafted chains against the target's probabilities, from given random numbers.
``slots``       :func:`jetspec_b200.ops.plan_slots`: pages granted, slot maps and the rows of a forward made from request lengths.

The plain forms are elementary torch operations: attention in 32 bits, probabilities, running sums and their comparisons in 64.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 16               # the engine's default page
SPREAD, SHIFT = 3.0, 0.75      # logits of a draft head, and how far the target's are from them
ACCEPTED = 0.71         # the share of drafts that is then accepted


def listed():
    return [
        # eight samples of one short chat prompt, a token each: the smallest attention, launches and latency count
        dict(name="attention_decode_8", kind="attention", heads=32, kv_heads=8, n=8, prefix=1024, lo=1, hi=64, q_lo=1, q_hi=1,
             form="tree"),
        # 64 users behind one long system prompt, a token each
        dict(name="attention_decode_64", kind="attention", heads=32, kv_heads=8, n=64, prefix=8192, lo=16, hi=512, q_lo=1, q_hi=1,
             form="causal"),
        # 32 questions about one book, many query heads
        dict(name="attention_decode_book", kind="attention", heads=64, kv_heads=8, n=32, prefix=65536, lo=5, hi=300, q_lo=1, q_hi=1,
             form="causal"),
        # a verify forward: 16 token trees of 128 nodes behind a long prompt
        dict(name="attention_trees_16", kind="attention", heads=32, kv_heads=8, n=16, prefix=8192, lo=0, hi=500, q_lo=128, q_hi=128,
             form="tree"),
        # the users' own prompts behind the system prompt, ragged, a prefix that ends inside a page
        dict(name="attention_portions", kind="attention", heads=32, kv_heads=4, n=6, prefix=2501, lo=0, hi=700, q_lo=33, q_hi=901,
             form="causal"),
        # one request, three drafts
        dict(name="verify_1", kind="verify", vocab=151936, n=1, lo=3, hi=3, dtype="fp32", each=False),
        # a batch on half the bytes, a temperature of its own for each request
        dict(name="verify_16", kind="verify", vocab=151936, n=16, lo=2, hi=8, dtype="bf16", each=True),
        # a small vocabulary of odd size, short chains
        dict(name="verify_small_vocab", kind="verify", vocab=32001, n=48, lo=0, hi=5, dtype="fp32", each=False),
        # a full batch, long chains
        dict(name="verify_64", kind="verify", vocab=151936, n=64, lo=4, hi=16, dtype="fp32", each=False),
        # a decode step of 16 requests: one row each, now and then a page
        dict(name="slots_decode_16", kind="slots", page=16, n=16, lo=30, hi=4000, q_lo=1, q_hi=1, window=0),
        # a verify step of 128 requests: 128 rows each, trees' windows mapped before
        dict(name="slots_trees_128", kind="slots", page=16, n=128, lo=100, hi=8000, q_lo=128, q_hi=128, window=64),
        # 256 whole prompts admitted at once
        dict(name="slots_prompts_256", kind="slots", page=16, n=256, lo=0, hi=0, q_lo=50, q_hi=16000, window=0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "verify", "slots"])
    if kind == "attention":
        heads, kv = rng.choice([(32, 8), (32, 4), (16, 8), (64, 8)])
        form = rng.choice(["decode", "tree", "causal"])
        n = _spread(rng, 1, 64 if form == "decode" else 16)
        q_hi = 1 if form == "decode" else _spread(rng, 2, 256 if form == "tree" else 900)
        q_hi = max(1, min(q_hi, 2048 // n))
        prefix = _spread(rng, 50, 32768 if form == "decode" else 8192)
        if heads == 64:
            q_hi, prefix = (q_hi + 1) // 2, (prefix + 1) // 2
        return dict(kind=kind, heads=heads, kv_heads=kv, n=n, prefix=prefix, lo=rng.randint(0, 40), hi=_spread(rng, 40, 500),
                    q_lo=1 if form == "decode" else rng.randint(1, q_hi), q_hi=q_hi, form="causal" if form == "decode" else form)
    if kind == "verify":
        lo = rng.randint(0, 4)
        return dict(kind=kind, vocab=_spread(rng, 1000, 151936), n=_spread(rng, 1, 64), lo=lo, hi=rng.randint(max(1, lo), 16),
                    dtype=rng.choice(["fp32", "bf16"]), each=rng.random() < 0.5)
    q_lo = 1 if rng.random() < 0.5 else _spread(rng, 2, 400)
    q_hi = q_lo if q_lo == 1 else _spread(rng, q_lo, 16000)
    return dict(kind=kind, page=rng.choice([16, 16, 32, 64]), n=_spread(rng, 1, 256), lo=rng.randint(0, 100), hi=_spread(rng, 100, 8000),
                q_lo=q_lo, q_hi=q_hi, window=rng.choice([0, 0, 16, 100]))


# ------------------------------------------------------------------ inputs
def _even(lo, hi, n):
    """``n`` lengths from ``lo`` to ``hi``, evenly apart."""
    return [(lo + hi + 1) // 2] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(lo, hi, n, gen):
    """The same in an order of the seed's."""
    return torch.tensor(_even(lo, hi, n), device="cuda")[torch.randperm(n, generator=gen, device="cuda")]


def _offsets(counts):
    return torch.cat((counts.new_zeros(1), counts.cumsum(0)))


def _i32(t):
    return t.to(torch.int32).contiguous()


def _tree_bits(counts, most, words, gen):
    """Ancestor-or-self bits of random trees: every node hangs below one of the few before it."""
    n = counts.numel()
    node = torch.arange(most, device="cuda")
    back = 1 + (torch.rand(n, most, generator=gen, device="cuda") * 6).long()
    parent = (node - back).clamp_min(0)
    seen = torch.eye(most, device="cuda").expand(n, most, most).clone()
    seen.scatter_(2, parent[..., None], 1.0)
    for _ in range(max(1, most - 1).bit_length()):          # paths of twice the length each time
        seen = ((seen @ seen) > 0).float()
    seen = torch.nn.functional.pad(seen, (0, words * 32 - most)).view(n, most, words, 32).long()
    bits = (seen << torch.arange(32, device="cuda")).sum(-1)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits)
    return _i32(bits[node[None, :] < counts[:, None]])


def _prepare_attention(case, gen):
    n, hq, hkv, prefix = case["n"], case["heads"], case["kv_heads"], case["prefix"]
    counts, behind = _lengths(case["q_lo"], case["q_hi"], n, gen), _lengths(case["lo"], case["hi"], n, gen)
    past = prefix + behind
    most = prefix + case["hi"] + case["q_hi"]
    columns = -(-most // PAGE)
    shared, whole = -(-prefix // PAGE), prefix // PAGE
    pages = torch.randperm(shared + n * (columns - whole), generator=gen, device="cuda")
    table = torch.empty(n, columns, dtype=torch.long, device="cuda")
    table[:, :whole] = pages[:whole]
    table[:, whole:] = pages[shared:].view(n, columns - whole)       # the page in which the prefix ends is every sequence's own ...
    pos = torch.arange(columns * PAGE, device="cuda")
    slot_map = table[:, pos // PAGE] * PAGE + pos % PAGE
    slot_map[:, :prefix] = pages[pos[:prefix] // PAGE] * PAGE + pos[:prefix] % PAGE      # ... but for the prefix's own positions
    slots = pages.numel() * PAGE
    rows = int(counts.sum())
    make = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    return dict(kind="attention", q=make(rows, hq, 128) * 1.5, k=make(hkv, slots, 128), v=make(hkv, slots, 128), slot_map=_i32(slot_map),
                seq_rows=_i32(torch.arange(n, device="cuda")), cu_q=_i32(_offsets(counts)), past=_i32(past), scale=128 ** -0.5,
                bits=_tree_bits(counts, case["q_hi"], -(-case["q_hi"] // 32), gen) if case["form"] == "tree" else None,
                causal=case["form"] == "causal", prefix=prefix, max_q=case["q_hi"], max_keys=int((past + counts).max()))


def _prepare_verify(case, gen):
    n, vocab = case["n"], case["vocab"]
    counts = _lengths(case["lo"], case["hi"], n, gen)
    cu = _offsets(counts)
    drafted = int(cu[-1])
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    draft = (torch.randn(drafted, vocab, generator=gen, device="cuda") * SPREAD).to(dtype)
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), counts)
    target = torch.randn(drafted + n, vocab, generator=gen, device="cuda") * SPREAD
    at = torch.arange(drafted, device="cuda") + seq
    target[at] = draft.float() + SHIFT * target[at] / SPREAD
    rand = lambda k: torch.rand(k, generator=gen, device="cuda")
    temperature = 0.7 + 0.5 * rand(n) if case["each"] else 1.0
    hot = temperature[seq, None] if case["each"] else 1.0
    weights = (draft.float() / hot).softmax(-1)
    drafts = torch.searchsorted(weights.cumsum(-1), rand(drafted)[:, None]).clamp_max(vocab - 1).view(-1)
    return dict(kind="verify", target=target.to(dtype), draft=draft, drafts=_i32(drafts), cu=_i32(cu), u=rand(drafted), v=rand(n),
                temperature=temperature, most=case["hi"])


def _prepare_slots(case, gen):
    n, page = case["n"], case["page"]
    past, counts = _lengths(case["lo"], case["hi"], n, gen), _lengths(case["q_lo"], case["q_hi"], n, gen)
    mapped = past + case["window"]
    most = case["hi"] + max(case["q_hi"], case["window"]) + page
    columns = -(-most // page)
    need = (-(-(past + counts) // page) - -(-mapped // page)).clamp_min(0)
    total = int(need.sum())
    pages = torch.randperm(n * columns + total, generator=gen, device="cuda")
    pos = torch.arange(columns * page, device="cuda")
    slot_map = pages[total:].view(n, columns)[:, pos // page] * page + pos % page
    slot_map = torch.where(pos < (-(-mapped // page) * page)[:, None], slot_map, 0)
    return dict(kind="slots", past=_i32(past), counts=_i32(counts), mapped=_i32(mapped),
                seq_rows=_i32(torch.randperm(n, generator=gen, device="cuda")), free=_i32(pages[:total]), page=page,
                slot_map=_i32(slot_map), rows=int(counts.sum()))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"attention": _prepare_attention, "verify": _prepare_verify, "slots": _prepare_slots}[case["kind"]](case, gen)


# ------------------------------------------------------------------ plain forms
def _attention(s):
    """The prefix's scores of all rows at once beside those of the sequences' own keys, padded to the longest."""
    q, cu, past, prefix = s["q"].float(), s["cu_q"].long(), s["past"].long(), s["prefix"]
    rows, hq, dim = q.shape
    hkv = s["k"].shape[0]
    counts = cu[1:] - cu[:-1]
    i, m = torch.arange(s["max_q"], device=q.device), torch.arange(s["max_keys"] - prefix, device=q.device)
    n = counts.numel()
    at = (cu[:-1, None] + i).clamp_max(rows - 1)
    qb = q[at].view(n, i.numel(), hkv, hq // hkv, dim) * s["scale"]
    slots = s["slot_map"].long()[s["seq_rows"].long()]
    kp, vp = (s[x][:, slots[0, :prefix]].float() for x in "kv")
    ks, vs = (s[x][:, slots[:, prefix:s["max_keys"]]].float() for x in "kv")
    j = prefix + m - past[:, None]                                   # place among the new rows, below 0: committed
    if s["causal"]:
        seen = j[:, None, :] <= i[:, None]
    else:
        bits = s["bits"].long()[at]
        word = (j // 32).clamp(0, bits.shape[-1] - 1)[:, None, :].expand(n, i.numel(), m.numel())
        seen = (j < 0)[:, None, :] | ((bits.gather(2, word) >> (j % 32)[:, None, :]) & 1).bool()
    seen = seen & (j < counts[:, None])[:, None, :]
    sp = torch.einsum("bnhgd,hpd->bhgnp", qb, kp)
    ss = torch.einsum("bnhgd,hbmd->bhgnm", qb, ks).masked_fill(~seen[:, None, None], -math.inf)
    top = torch.maximum(sp.amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
    sp, ss = (sp - top).exp(), (ss - top).exp()
    out = torch.einsum("bhgnp,hpd->bnhgd", sp, vp) + torch.einsum("bhgnm,hbmd->bnhgd", ss, vs)
    out = out / (sp.sum(-1) + ss.sum(-1)).permute(0, 3, 1, 2)[..., None]
    return out.reshape(n, i.numel(), hq * dim)[i < counts[:, None]].to(s["q"].dtype)


def _probabilities(logits, temperature):
    x = logits.double() / temperature
    x = (x - x.amax(-1, keepdim=True)).exp()
    return x / x.sum(-1, keepdim=True)


def _verify(s):
    cu, drafts = s["cu"].long(), s["drafts"].long()
    counts = cu[1:] - cu[:-1]
    n, drafted = counts.numel(), drafts.numel()
    t = torch.arange(drafted, device=drafts.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    hot = s["temperature"].double()[:, None] if torch.is_tensor(s["temperature"]) else s["temperature"]
    each = hot[seq] if torch.is_tensor(hot) else hot
    p, q = _probabilities(s["target"][t + seq], each), _probabilities(s["draft"], each)
    good = s["u"].double() * q.gather(1, drafts[:, None])[:, 0] < p.gather(1, drafts[:, None])[:, 0]
    wide = torch.arange(max(1, s["most"]), device=drafts.device)
    padded = torch.cat((good, good.new_zeros(1)))[(cu[:-1, None] + wide).clamp_max(drafted)] & (wide < counts[:, None])
    accepted = padded.long().cumprod(1).sum(1)
    weight = _probabilities(s["target"][cu[:-1] + torch.arange(n, device=drafts.device) + accepted], hot)
    if drafted:
        left = (weight - _probabilities(s["draft"][(cu[:-1] + accepted).clamp_max(drafted - 1)], hot)).clamp_min(0)
        weight = torch.where((accepted < counts)[:, None], left, weight)
    run = weight.cumsum(-1)
    token = (run <= s["v"].double()[:, None] * run[:, -1:]).sum(-1)
    return accepted.to(torch.int32), token


def _slots(s):
    past, counts, page, slot_map = s["past"].long(), s["counts"].long(), s["page"], s["slot_map"]
    held = -(-s["mapped"].long() // page)
    need = (-(-(past + counts) // page) - held).clamp_min(0)
    cu_q, cu_pages = _offsets(counts), _offsets(need)
    free = s["free"].long()
    pos = torch.arange(slot_map.shape[1], device=past.device)
    k = pos // page - held[:, None]
    new = free[(cu_pages[:-1, None] + k).clamp(0, max(0, free.numel() - 1))] * page + pos % page if free.numel() else pos.expand(k.shape)
    rows = s["seq_rows"].long()
    slot_map[rows] = torch.where((k >= 0) & (k < need[:, None]), new, slot_map[rows].long()).to(torch.int32)
    t = torch.arange(s["rows"], device=past.device)
    seq = torch.searchsorted(cu_q[1:].contiguous(), t, right=True)
    positions = past[seq] + t - cu_q[seq]
    return _i32(cu_q), _i32(positions), slot_map[rows[seq], positions], _i32(cu_pages), slot_map


def run(state):
    s = state
    if own:
        from jetspec_b200 import ops
        if s["kind"] == "attention":
            return ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["slot_map"], s["seq_rows"], s["cu_q"], s["past"], s["bits"],
                                               s["scale"], s["prefix"], causal=s["causal"], max_q=s["max_q"])
        if s["kind"] == "verify":
            return ops.verify_chains(s["target"], s["draft"], s["drafts"], s["cu"], s["u"], s["v"], temperature=s["temperature"])
        return (*ops.plan_slots(s["past"], s["counts"], s["seq_rows"], s["free"], s["page"], s["slot_map"], s["rows"],
                                mapped_lens=s["mapped"]), s["slot_map"])
    return {"attention": _attention, "verify": _verify, "slots": _slots}[s["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n = case["n"]
    if case["kind"] == "attention":
        hq, hkv, prefix = case["heads"], case["kv_heads"], case["prefix"]
        counts = _even(case["q_lo"], case["q_hi"], n)
        rows, committed, new = sum(counts), sum(_even(case["lo"], case["hi"], n)), sum(counts)
        keys = sum(c * (prefix + (case["lo"] + case["hi"]) / 2 + (c + 1) / 2) for c in counts)        # a tree's mask is not known here
        kv = 4 * hkv * 128 * (prefix + committed + new)
        return {"bytes": kv + 2 * 2 * rows * hq * 128 + 4 * (prefix + committed + new), "flops": 4 * 128 * hq * keys}
    if case["kind"] == "verify":
        # the rows up to the first rejection; the last ones are summed and searched
        size = 4 if case["dtype"] == "fp32" else 2
        counts = _even(case["lo"], case["hi"], n)
        target = sum(sum(ACCEPTED ** i for i in range(c + 1)) for c in counts)
        draft = sum(sum(ACCEPTED ** i for i in range(c)) for c in counts)
        return {"bytes": (target + draft) * case["vocab"] * size, "flops": 4 * (target + draft) * case["vocab"]}
    page, counts = case["page"], _even(case["q_lo"], case["q_hi"], n)
    rows = sum(counts)
    new = max(0, rows - case["window"] * n)
    return {"bytes": 20 * n + 4 * new / page + 4 * new + 8 * rows, "flops": rows + new}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Attention, sequence by sequence.  The others answer in whole numbers."""
    if case["kind"] != "attention":
        return None
    s = prepare(case, seed)
    hkv = s["k"].shape[0]
    g = s["q"].shape[1] // hkv
    out = []
    cu, past, seq_rows = s["cu_q"].tolist(), s["past"].tolist(), s["seq_rows"].tolist()
    for b, row in enumerate(seq_rows):
        c, total = cu[b + 1] - cu[b], past[b] + cu[b + 1] - cu[b]
        slots = s["slot_map"][row, :total].long()
        if s["causal"]:
            new = torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
        else:
            j = torch.arange(c, device="cuda")
            new = ((s["bits"][cu[b]:cu[b + 1]].long()[:, j // 32] >> (j % 32)) & 1) == 1
        seen = torch.cat((torch.ones(c, past[b], dtype=torch.bool, device="cuda"), new), 1)
        heads = []
        for h in range(hkv):
            k, v = s["k"][h, slots].double(), s["v"][h, slots].double()
            x = s["q"][cu[b]:cu[b + 1], h * g:(h + 1) * g].double().transpose(0, 1) @ k.T * s["scale"]
            heads.append(torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v)
        out.append(torch.cat(heads).transpose(0, 1).reshape(c, -1))
    return torch.cat(out)
