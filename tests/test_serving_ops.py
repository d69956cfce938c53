"""Operators of a batched serving step: slot planning, attention behind a shared prefix, verification of drafted chains.

On the CPU the PyTorch implementations against plain loops; on the GPU the kernels against them, in 64 bits where they compute.
"""
import math
import random

import pytest
import torch

from jetspec_b200 import ops
from jetspec_b200.ops import reference as ref

gpu = pytest.mark.gpu
I32 = torch.int32


@pytest.fixture
def clean():
    """The device's status word is clear before and after."""
    from jetspec_b200.ops import cuda_ext
    cuda_ext.check_status("cuda")
    yield cuda_ext
    cuda_ext.check_status("cuda")


def i32(*v, device="cpu"):
    return torch.tensor(v, dtype=I32, device=device)


# ------------------------------------------------------------------ slot planning
def plan_by_loops(past, counts, rows, free, page, slot_map, T, mapped):
    """The contract of ``plan_slots``, request by request."""
    free, out, taken, cu_q, cu_p = list(free), [], set(), [0], [0]
    slot_map = [list(r) for r in slot_map]
    max_len = len(slot_map[0])
    for p, c, r, m in zip(past, counts, rows, mapped):
        sound = 0 <= r < len(slot_map) and r not in taken
        taken.add(r)
        held, want = -(-m // page), -(-(p + c) // page)
        pages = {j: free.pop(0) if free else -1 for j in range(held, want)}
        slot = lambda pos: -1 if pages[pos // page] < 0 else pages[pos // page] * page + pos % page
        for pos in range(held * page, want * page):
            if sound and pos < max_len:
                slot_map[r][pos] = slot(pos)
        for pos in range(p, p + c):
            out.append((pos, -1 if not sound or pos >= max_len else slot_map[r][pos]))
        cu_q.append(cu_q[-1] + c)
        cu_p.append(cu_p[-1] + max(0, want - held))
    out = (out + [(0, -1)] * T)[:T]
    return cu_q, [o[0] for o in out], [o[1] for o in out], cu_p, slot_map


def plan_case(seed, B, page, max_len, count, window=0, short=0, extra_rows=0, device="cpu"):
    """Requests of mixed lengths on random pages; ``short``: how many pages are missing."""
    r = random.Random(seed)
    past = [r.randint(0, max(0, max_len - count - page)) for _ in range(B)]
    counts = [r.choice([0, 1, count, r.randint(0, count)]) for _ in range(B)]
    mapped = [min(p + r.choice([0, window]), max_len) for p in past]
    seqs = B + 2
    need = sum(max(0, -(-(p + c) // page) - -(-m // page)) for p, c, m in zip(past, counts, mapped))
    ids = list(range(need + seqs))
    r.shuffle(ids)
    g = torch.Generator().manual_seed(seed)
    slot_map = torch.randint(0, 1000, (seqs, max_len), generator=g, dtype=I32)
    rows = r.sample(range(seqs), B)
    t = lambda v: torch.tensor(v, dtype=I32, device=device)
    return dict(past_lens=t(past), counts=t(counts), seq_rows=t(rows), free_pages=t(ids[:max(0, need - short)]), page_size=page,
                slot_map=slot_map.to(device), rows=sum(counts) + extra_rows, mapped_lens=t(mapped))


PLANS = [  # B, page, max_len, count, window, missing pages, rows too many (below 0: too few)
    (1, 16, 64, 1, 0, 0, 0), (1, 16, 64, 40, 0, 0, 3), (7, 16, 200, 33, 20, 0, 5), (16, 1, 50, 9, 3, 0, 0), (33, 5, 121, 60, 7, 0, 1),
    (9, 64, 512, 130, 0, 0, 0), (5, 16, 160, 50, 0, 4, 2), (300, 16, 96, 20, 16, 0, 7), (6, 128, 100, 30, 0, 0, 4),
]


def run_plan(fn, case):
    c = dict(case)
    slot_map = c["slot_map"].clone()
    out = fn(c["past_lens"], c["counts"], c["seq_rows"], c["free_pages"], c["page_size"], slot_map, c["rows"], c["mapped_lens"])
    return [o.tolist() for o in out] + [slot_map.tolist()]


def plan_expected(case):
    c = {k: v.tolist() if torch.is_tensor(v) else v for k, v in case.items()}
    return list(plan_by_loops(c["past_lens"], c["counts"], c["seq_rows"], c["free_pages"], c["page_size"], c["slot_map"], c["rows"],
                              c["mapped_lens"]))


@pytest.mark.parametrize("plan", PLANS)
def test_plan_slots_by_loops(plan):
    B, page, max_len, count, window, short, more = plan
    case = plan_case(B + page, B, page, max_len, count, window, short, more)
    assert run_plan(ops.plan_slots, case) == plan_expected(case)


def odd_plans(device="cpu"):
    """Calls with something wrong in them, and what the status word says: (case, status)."""
    def case(past, counts, rows, free, page, max_len, T, seqs=3):
        t = lambda v: torch.tensor(v, dtype=I32, device=device)
        return dict(past_lens=t(past), counts=t(counts), seq_rows=t(rows), free_pages=t(free), page_size=page,
                    slot_map=torch.arange(seqs * max_len, dtype=I32, device=device).view(seqs, max_len) + 500, rows=T, mapped_lens=t(past))
    return [
        (case([5, 9], [4, 4], [1, 1], [3, 4], 4, 32, 8), 5),          # the same slot-map row twice: the second gets nothing
        (case([5, 9], [4, 4], [1, 7], [3, 4], 4, 32, 8), 5),          # a row out of range
        (case([5, 9], [4, 4], [-1, 0], [3, 4], 4, 32, 8), 5),
        (case([30, 2], [6, 1], [0, 1], [3, 4], 4, 32, 7), 5),         # positions past the slot map
        (case([4, 4], [4, 4], [0, 1], [3], 4, 32, 8), 13),            # too few pages
        (case([4, 4], [4, 4], [0, 1], [], 4, 32, 8), 13),
        (case([4, 4], [4, 4], [0, 1], [3, 4], 4, 32, 6), 14),         # too few rows
    ]


def test_plan_slots_with_something_wrong():
    for case, _ in odd_plans():
        assert run_plan(ops.plan_slots, case) == plan_expected(case)


def test_plan_slots_of_nothing():
    for device in ["cpu"] + ["cuda"] * torch.cuda.is_available():
        e = torch.empty(0, dtype=I32, device=device)
        slot_map = torch.full((2, 8), 7, dtype=I32, device=device)
        cu_q, positions, slots, cu_pages = ops.plan_slots(e, e, e, e, 4, slot_map, 3)
        assert cu_q.tolist() == [0] and cu_pages.tolist() == [0] and positions.tolist() == [0] * 3 and slots.tolist() == [-1] * 3
        assert [o.numel() for o in ops.plan_slots(e, e, e, e, 4, slot_map, 0)] == [1, 0, 0, 1] and bool((slot_map == 7).all())


@gpu
@pytest.mark.parametrize("plan", PLANS + [(3, 16, 70000, 66000, 0, 0, 11), (1000, 16, 300, 40, 0, 0, 0)])
def test_plan_slots_kernel(clean, plan):
    B, page, max_len, count, window, short, more = plan
    case = plan_case(B + page, B, page, max_len, count, window, short, more, device="cuda")
    cpu = {k: v.cpu() if torch.is_tensor(v) else v for k, v in case.items()}
    assert run_plan(ops.plan_slots, case) == run_plan(ref.plan_slots, cpu)
    if short:
        with pytest.raises(RuntimeError, match="free pages ran out"):
            clean.check_status("cuda")


@gpu
def test_plan_slots_kernel_with_something_wrong(clean):
    for (case, status), (cpu, _) in zip(odd_plans("cuda"), odd_plans()):
        assert run_plan(ops.plan_slots, case) == run_plan(ref.plan_slots, cpu)
        with pytest.raises(RuntimeError, match=f"status {status}"):
            clean.check_status("cuda")


def kernel_refuses(call, *words):
    with pytest.raises(ValueError, match="|".join(words)):
        call()


def test_plan_slots_refusals():
    from jetspec_b200.ops import cuda_ext
    z, m = i32(0, 0), torch.zeros(2, 8, dtype=I32)
    plan = lambda **kw: cuda_ext.plan_slots(**{**dict(past_lens=z, counts=z, seq_rows=z, free_pages=z, page_size=4, slot_map=m, rows=2), **kw})
    kernel_refuses(lambda: plan(past_lens=z.long()), "past_lens")
    kernel_refuses(lambda: plan(free_pages=i32(1, 2, 3, 4)[::2]), "free_pages")
    kernel_refuses(lambda: plan(slot_map=torch.zeros(8, 2, dtype=I32).t()), "slot_map")
    kernel_refuses(lambda: plan(counts=i32(0)), "length")
    kernel_refuses(lambda: plan(mapped_lens=i32(0)), "length")
    kernel_refuses(lambda: plan(page_size=0), "page_size")
    kernel_refuses(lambda: plan(rows=-1), "rows")


# ------------------------------------------------------------------ verification of chains
def chains(seed, lens, V, dtype=torch.float32, spread=3.0, shift=0.75, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    D, B = sum(lens), len(lens)
    draft = (torch.randn(D, V, generator=g) * spread).to(dtype)
    target = torch.randn(D + B, V, generator=g) * spread
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(lens, dtype=torch.long))
    at = torch.arange(D) + seq
    target[at] = draft.float() + shift * target[at] / spread
    drafts = torch.multinomial(draft.float().softmax(-1), 1, generator=g).view(-1).to(I32) if D else torch.zeros(0, dtype=I32)
    cu = torch.tensor([0] + torch.tensor(lens, dtype=torch.long).cumsum(0).tolist(), dtype=I32)
    out = dict(target_logits=target.to(dtype), draft_logits=draft, drafts=drafts, cu_drafts=cu, accept_u=torch.rand(D, generator=g),
               sample_u=torch.rand(B, generator=g))
    return {k: v.to(device) for k, v in out.items()}


def test_verify_chains_keeps_the_targets_distribution():
    """20000 chains of two drafts over 6 tokens: the first token kept is distributed like the target's first row, and the second, after
    an accepted first, like the target's second row.  Bounds: 4.5 standard deviations of a share of n draws."""
    n, V = 20000, 6
    one = chains(0, [2], V, spread=1.0, shift=1.5)
    g = torch.Generator().manual_seed(1)
    q, p = one["draft_logits"].softmax(-1), one["target_logits"].softmax(-1)
    drafts = torch.stack([torch.multinomial(q[i], n, replacement=True, generator=g) for i in range(2)], 1)
    kept, token = ref.verify_chains(one["target_logits"].repeat(n, 1), one["draft_logits"].repeat(n, 1), drafts.reshape(-1).to(I32),
                                    torch.arange(n + 1, dtype=I32) * 2, torch.rand(2 * n, generator=g), torch.rand(n, generator=g))
    first = torch.where(kept > 0, drafts[:, 0], token)
    second = torch.where(kept > 1, drafts[:, 1], token)[kept > 0]
    for got, want in ((first, p[0]), (second, p[1])):
        share = torch.bincount(got, minlength=V) / got.numel()
        assert bool(((share - want).abs() <= 4.5 * (want * (1 - want) / got.numel()).sqrt()).all())
    assert 0.2 < float((kept > 0).double().mean()) < 0.95


def test_verify_chains_by_hand():
    """Point masses and empty rows, where every number is known."""
    inf = math.inf
    row = lambda *p: torch.tensor([math.log(x) if x else -inf for x in p])
    call = lambda target, draft, x, u, v, **kw: tuple(int(t) for t in ops.verify_chains(
        torch.stack(target), torch.stack(draft), i32(*x), i32(0, len(x)), torch.tensor(u), torch.tensor([v]), **kw))
    p, q = row(.5, .25, .25), row(.25, .5, .25)
    assert call([p, p], [q], [1], [.49], .0) == (1, 0)                # u q < p: .49 * .5 < .25; then the first of the last row
    assert call([p, p], [q], [1], [.51], .9) == (0, 0)                # only token 0 is in the difference
    assert call([p, row(0, 0, 1)], [q], [1], [.4], .9) == (1, 2)
    assert call([row(0, .5, .5), p], [q], [0], [.0], .0) == (0, 2)    # the target gives the draft nothing: 0 < 0 is false; .25 is left at 2
    empty = row(0, 0, 0)
    assert call([empty, p], [q], [1], [.0], .5) == (0, -1)            # a row whose mask leaves nothing
    assert call([p, empty], [q], [0], [.5], .5) == (1, -1)
    assert call([p, p], [empty], [2], [.9], .3) == (1, 0)             # the draft's row says nothing: whatever the target can say is kept
    assert call([p, p], [q], [1], [.9], .7, temperature=0.0) == (0, 0)
    assert call([p, p], [p], [0], [.9], .7, temperature=0.0) == (1, 0)
    assert call([p, row(.25, .375, .375)], [p], [0], [.9], .7, temperature=0.0) == (1, 1)      # equal: the lowest index
    assert call([p, p], [p], [0], [.6], .4, draft_temperature=0.0) == (0, 1)      # drafted for certain, .6 >= .5: without token 0
    assert call([p, p], [q], [7], [.0], .0) == (0, 0)                 # no such token


CHAINS = [([3], 151936, torch.float32), ([0], 1000, torch.float32), ([1], 1, torch.float32), ([2, 0, 5, 1], 7, torch.bfloat16),
          ([4] * 20, 32001, torch.float32), ([6, 3, 0, 8, 2], 151936, torch.bfloat16), ([1, 2] * 150, 515, torch.float32),
          ([40], 4099, torch.bfloat16), (list(range(17)), 50001, torch.float32), ([700, 1], 33, torch.float32)]


@gpu
@pytest.mark.parametrize("lens,V,dtype", CHAINS)
def test_verify_chains_kernel(clean, lens, V, dtype):
    c = chains(len(lens) + V, lens, V, dtype)
    dev = {k: v.cuda() for k, v in c.items()}
    hot = 0.5 + torch.rand(len(lens), generator=torch.Generator().manual_seed(3))
    cold = hot.clone()
    cold[::2] = 0.0
    for kw in (dict(), dict(temperature=0.7), dict(temperature=hot, draft_temperature=1.0), dict(temperature=cold), dict(temperature=0.0),
               dict(draft_temperature=0.0)):
        want = ref.verify_chains(**c, **kw)
        got = ops.verify_chains(**dev, **{k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()})
        assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
        assert got[0].dtype == I32 and got[1].dtype == torch.int64


@gpu
@pytest.mark.parametrize("lens,shift", [([0, 1, 2, 3, 4, 5, 8, 9, 10, 12, 17, 30, 40], 0.05), ([1] * 100 + [0, 2], 0.75)])
def test_verify_chains_kernel_of_many_rows(clean, lens, shift):
    """Chains that are kept for long, many that are short, over a large vocabulary: the same result whenever blocks come to their rows."""
    c = chains(1, lens, 151936, shift=shift)
    dev = {k: v.cuda() for k, v in c.items()}
    want = ref.verify_chains(**c)
    for _ in range(3):
        got = ops.verify_chains(**dev)
        assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()


@gpu
def test_verify_chains_kernel_masked_and_strided(clean):
    """Vocabularies cut down to a few tokens (-inf elsewhere), empty rows, views of wider matrices, rows off 16-byte boundaries, drafts
    with the same token again, numbers at the ends of [0, 1)."""
    for V, dtype in ((1000, torch.float32), (1003, torch.bfloat16), (9001, torch.float16)):
        c = chains(V, [5, 1, 0, 7, 3, 2], V, dtype)
        g = torch.Generator().manual_seed(9)
        keep = torch.rand(1, V, generator=g) < 0.02
        keep[0, c["drafts"].long()[::2]] = True
        for name in ("target_logits", "draft_logits"):
            c[name] = c[name].masked_fill(~keep, -math.inf)
        c["target_logits"][3] = -math.inf
        c["draft_logits"][9] = -math.inf
        c["drafts"][6:10] = c["drafts"][6]
        c["accept_u"][0], c["accept_u"][6], c["sample_u"][0], c["sample_u"][1] = 0.0, 1 - 2 ** -24, 0.0, 1 - 2 ** -24
        want = ref.verify_chains(**c)
        dev = {k: v.cuda() for k, v in c.items()}
        wide = {k: torch.full((dev[k].shape[0], V + 5), math.nan, dtype=dtype, device="cuda") for k in ("target_logits", "draft_logits")}
        for k, w in wide.items():
            w[:, 3:V + 3] = dev[k]
            dev[k] = w[:, 3:V + 3]
        got = ops.verify_chains(**dev)
        assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()


@gpu
def test_verify_chains_kernel_bad_token(clean):
    c = chains(5, [3, 2], 100, device="cuda")
    c["drafts"][0], c["drafts"][4], c["accept_u"] = -1, 100, c["accept_u"] * 0
    accepted, token = ops.verify_chains(**c)
    assert accepted.tolist()[0] == 0 and accepted.tolist()[1] == 1 and bool((token >= 0).all() & (token < 100).all())
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        clean.check_status("cuda")


def test_verify_chains_refusals():
    from jetspec_b200.ops import cuda_ext
    c = chains(0, [2, 1], 9)
    call = lambda **kw: cuda_ext.verify_chains(**{**c, **kw})
    kernel_refuses(lambda: call(target_logits=c["target_logits"][:4]), "drafts of")
    kernel_refuses(lambda: call(draft_logits=c["draft_logits"][:, :8]), "drafts of")
    kernel_refuses(lambda: call(drafts=c["drafts"].long()), "drafts")
    kernel_refuses(lambda: call(accept_u=c["accept_u"].double()), "accept_u")
    kernel_refuses(lambda: call(sample_u=c["sample_u"][:1]), "sample_u")
    kernel_refuses(lambda: call(temperature=-1.0), "temperature")
    kernel_refuses(lambda: call(temperature=torch.ones(3)), "temperature")
    kernel_refuses(lambda: call(draft_temperature=torch.ones(2, dtype=torch.float64)), "draft_temperature")


# ------------------------------------------------------------------ attention behind a shared prefix
def tree_bits(counts, gen, words):
    """Ancestor bits of random trees; some rows see nothing of their tree, not even themselves."""
    rows = []
    for n in counts:
        seen = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            if i:
                seen[i] = seen[int(torch.randint(max(0, i - 7), i, (1,), generator=gen))]
            seen[i, i] = True
        seen[torch.rand(n, generator=gen) < 0.1] = False
        rows.append(ref.pack_ancestor_bits(seen, words))
    return torch.cat(rows) if rows else torch.zeros(0, words, dtype=I32)


def attention_case(seed, heads, kv_heads, prefix, behind, counts, causal, page=16, dim=128, dtype=torch.bfloat16, device="cpu",
                   more_rows=0, slack=2.0):
    """A pool of random pages whose first ``prefix`` positions all sequences share; slots that no position uses hold NaN."""
    g = torch.Generator().manual_seed(seed)
    B, T = len(counts), sum(counts) + more_rows
    most = prefix + max(b + c for b, c in zip(behind, counts)) + page
    columns, whole, shared = -(-most // page), prefix // page, -(-prefix // page)
    pages = torch.randperm(int(slack * (shared + B * columns)) + 1, generator=g)
    table = torch.empty(B, columns, dtype=torch.long)
    table[:, :whole] = pages[:whole]
    table[:, whole:] = pages[shared:shared + B * (columns - whole)].view(B, columns - whole)
    pos = torch.arange(columns * page)
    slot_map = table[:, pos // page] * page + pos % page
    slot_map[:, :prefix] = pages[pos[:prefix] // page] * page + pos[:prefix] % page
    for b in range(0, B, 2):          # a committed path trades slots inside a sequence
        n = prefix + behind[b]
        slot_map[b, prefix:n] = slot_map[b, prefix:n][torch.randperm(behind[b], generator=g)]
    S = pages.numel() * page
    used = torch.zeros(S, dtype=torch.bool)
    for b in range(B):
        used[slot_map[b, :prefix + behind[b] + counts[b]]] = True
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)
    pools = [make(kv_heads, S, dim) for _ in "kv"]
    for x in pools:
        x[:, ~used] = math.nan
    spare = torch.full((1, slot_map.shape[1]), S + 5)
    words = max(1, -(-max(counts) // 32)) + 1
    bits = None
    if not causal:
        bits = torch.cat((tree_bits(counts, g, words), torch.full((more_rows, words), -1, dtype=I32)))
    out = dict(q=make(T, heads, dim) * 1.5, k_pool=pools[0], v_pool=pools[1], slot_map=torch.cat((spare, slot_map)).to(I32),
               seq_rows=torch.arange(1, B + 1).to(I32), cu_q=torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=I32),
               past_lens=torch.tensor([prefix + b for b in behind], dtype=I32), mask_bits=bits, scale=dim ** -0.5, prefix_len=prefix, causal=causal)
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in out.items()}


def attention_exact(c):
    """The definition in 64 bits; rows that see no key, and rows behind the last sequence, are zero."""
    q, hkv = c["q"].double(), c["k_pool"].shape[0]
    T, hq, dim = q.shape
    out = torch.zeros(T, hq, dim, dtype=torch.float64, device=q.device)
    cu, past = c["cu_q"].tolist(), c["past_lens"].tolist()
    for b, row in enumerate(c["seq_rows"].tolist()):
        s, e = cu[b], cu[b + 1]
        slots = c["slot_map"][row, :past[b] + e - s].long()
        for i in range(s, e):
            own = torch.arange(e - s, device=q.device) <= i - s if c["causal"] else ref.unpack_ancestor_bits(c["mask_bits"][i:i + 1], e - s)[0]
            keys = slots[torch.cat((torch.ones(past[b], dtype=torch.bool, device=q.device), own))]
            if keys.numel():
                k, v = (c[x][:, keys].double().repeat_interleave(hq // hkv, 0) for x in ("k_pool", "v_pool"))
                out[i] = torch.einsum("hl,hld->hd", torch.softmax(torch.einsum("hd,hld->hl", q[i], k) * c["scale"], -1), v)
    return out.view(T, hq * dim)


def attend(c, **kw):
    return ops.shared_prefix_attention(c["q"], c["k_pool"], c["v_pool"], c["slot_map"], c["seq_rows"], c["cu_q"], c["past_lens"], c["mask_bits"],
                                       c["scale"], c["prefix_len"], causal=c["causal"], **kw)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("prefix,behind,counts", [(20, [0, 5, 3], [4, 1, 7]), (0, [0, 2], [3, 1]), (1, [0], [1]), (17, [2, 0, 0], [1, 0, 2])])
def test_shared_prefix_attention_by_definition(causal, prefix, behind, counts):
    c = attention_case(prefix, 4, 2, prefix, behind, counts, causal, page=4, dim=16, dtype=torch.float32, more_rows=2)
    assert torch.allclose(attend(c).double(), attention_exact(c), atol=1e-5)


# Rounding: probabilities become bf16 ahead of the second product (half a step is 2^-8 of each; they add up at random, and never to more than
# 2^-8 of the largest |v|, below 6 here, whatever the weights), the result once more (2^-8 of itself).  Sums and scores are fp32.
def attention_close(got, want, v_max=6.0):
    err = (got.double() - want).abs()
    assert bool((err <= 2 ** -8 * (v_max + want.abs())).all()), float(err.max())
    assert float(err.norm()) <= 5e-3 * float(want.norm()) + 1e-9


ATTENTION = [  # query heads, KV heads, prefix, committed behind it, new rows
    (32, 8, 1024, [3, 40, 17, 0], [1, 1, 1, 1]),
    (32, 8, 1000, [i * 7 % 90 for i in range(40)], [1] * 40),
    (8, 8, 300, [5], [1]),
    (16, 2, 130, [0, 1, 400], [16, 17, 15]),
    (12, 4, 257, [10, 0, 33], [40, 90, 3]),
    (10, 2, 77, [0, 200], [25, 26]),
    (64, 4, 128, [100, 3, 0, 9, 50], [8, 9, 1, 0, 30]),
    (4, 1, 1, [0, 0], [33, 1]),
    (32, 4, 0, [0, 130, 700], [70, 1, 128]),
    (2, 1, 5000, [0, 1], [2, 1]),
    (128, 1, 200, [7, 300], [3, 1]),
    (32, 8, 500, [20, 30, 0], [130, 0, 64]),
    (16, 8, 2000, [100] * 12, [3, 1, 2] * 4),
    (8, 1, 40, [9], [300]),
]


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,prefix,behind,counts", ATTENTION)
def test_shared_prefix_attention_kernel(clean, heads, kv, prefix, behind, counts, causal):
    c = attention_case(prefix + heads, heads, kv, prefix, behind, counts, causal, device="cuda", more_rows=3)
    want = attention_exact(c)
    got = attend(c, max_q=max(1, max(counts)))
    attention_close(got, want)
    attention_close(attend(c), want)      # without a bound on the rows


def test_shared_prefix_attention_refusals():
    from jetspec_b200.ops import cuda_ext
    c = attention_case(0, 4, 2, 20, [0, 5], [4, 3], False)
    call = lambda **kw: cuda_ext.shared_prefix_attention(**{**c, "max_q": 4, **kw})
    kernel_refuses(lambda: call(q=c["q"].float()), "q ")
    kernel_refuses(lambda: call(q=c["q"][..., :64]), "q ")
    kernel_refuses(lambda: call(k_pool=c["k_pool"][:, ::2]), "pools")
    kernel_refuses(lambda: call(v_pool=c["v_pool"].half()), "pools")
    kernel_refuses(lambda: call(q=c["q"][:, :3]), "heads")
    kernel_refuses(lambda: call(slot_map=c["slot_map"].long()), "slot_map")
    kernel_refuses(lambda: call(cu_q=c["cu_q"][:2]), "cu_q")
    kernel_refuses(lambda: call(mask_bits=None), "mask_bits")
    kernel_refuses(lambda: call(mask_bits=c["mask_bits"][:-1]), "mask_bits")
    kernel_refuses(lambda: call(prefix_len=-1), "prefix_len")
    kernel_refuses(lambda: call(prefix_len=c["slot_map"].shape[1] + 1), "prefix_len")
    kernel_refuses(lambda: call(max_q=-1), "max_q")
    kernel_refuses(lambda: call(scale=math.nan), "scale")
    kernel_refuses(lambda: call(out=torch.empty(7, 512)), "out")


@gpu
def test_shared_prefix_attention_of_odd_calls(clean):
    """A view of joint projections as queries, nothing to do, sequences without rows, a bound that is too low, slots that do not exist."""
    c = attention_case(1, 16, 4, 90, [0, 33, 7], [5, 0, 3], False, device="cuda")
    want = attention_exact(c)
    wide = torch.full((8, 24, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, :16] = c["q"]
    attention_close(attend({**c, "q": wide[:, :16]}), want)
    attention_close(attend({**c, "q": c["q"].transpose(0, 1).contiguous().transpose(0, 1)}), want)
    none = {k: c[k][:0] for k in ("q", "mask_bits", "seq_rows", "past_lens")}
    assert attend({**c, **none, "cu_q": i32(0, device="cuda")}).shape == (0, 16 * 128)
    assert not attend({**c, "cu_q": i32(0, 0, 0, 0, device="cuda")}, max_q=0).any()
    assert not attend({**c, "seq_rows": c["seq_rows"][:0], "past_lens": c["past_lens"][:0], "cu_q": i32(0, device="cuda")}).any()
    attend(c, max_q=4)
    with pytest.raises(RuntimeError, match="more new rows"):
        clean.check_status("cuda")
    attend({**attention_case(2, 8, 2, 64, [0, 0, 0, 0], [1, 1, 1, 1], True, device="cuda"), "past_lens": i32(64, 64, 47, 64, device="cuda")})
    with pytest.raises(RuntimeError, match="shorter than the prefix"):
        clean.check_status("cuda")
    for slot in (-1, c["k_pool"].shape[1]):
        m = c["slot_map"].clone()
        m[3, 95] = slot          # row 2 is the sequence without rows: nobody reads it
        attend({**c, "slot_map": m})
        with pytest.raises(RuntimeError, match="slot"):
            clean.check_status("cuda")


# ------------------------------------------------------------------ the three in a row
class Step:
    """Pages, rows and slots of a batch behind a shared prompt; its attention; what of its drafts the target keeps."""

    def __init__(self, device, prompt=37, lens=(5, 1, 8, 3), heads=8, kv=2, V=1009, dim=128):
        g = torch.Generator().manual_seed(11)
        B, T, page = len(lens), sum(lens), 16
        pages, shared = 12 * B, prompt // page * page
        put = lambda *s, dtype=torch.bfloat16: torch.randn(*s, generator=g).to(dtype).to(device)
        self.page, self.T, self.prefix = page, T, shared
        self.slot_map = torch.zeros(B + 1, 128, dtype=I32)
        self.slot_map[:, :shared] = torch.arange(shared, dtype=I32).flip(0)
        self.slot_map = self.slot_map.to(device)
        self.past, self.counts = (torch.tensor(v, dtype=I32, device=device) for v in ([prompt + 16 * b for b in range(B)], lens))
        self.mapped = torch.full((B,), shared, dtype=I32, device=device)
        self.rows = torch.arange(B, 0, -1, device=device).to(I32)
        self.free = (shared // page + torch.randperm(pages, generator=g)).to(I32).to(device)
        S = shared + pages * page
        self.k, self.v, self.q, self.knew, self.vnew = put(kv, S, dim), put(kv, S, dim), put(T, heads, dim), put(T, kv, dim), put(T, kv, dim)
        self.head = put(V, heads * dim, dtype=torch.float32) * 0.05
        self.draft = put(T - B, V, dtype=torch.float32)
        self.drafts = self.draft.argmax(-1).to(I32)
        self.cu_drafts = torch.tensor([0] + torch.tensor([n - 1 for n in lens]).cumsum(0).tolist(), dtype=I32, device=device)
        self.accept_u, self.sample_u = (torch.rand(n, generator=g).to(device) * 0.3 for n in (T - B, B))

    def __call__(self, o=ops):
        cu, positions, slots, cu_pages = o.plan_slots(self.past, self.counts, self.rows, self.free, self.page, self.slot_map, self.T,
                                                      mapped_lens=self.mapped)
        self.k[:, slots.long()], self.v[:, slots.long()] = self.knew.transpose(0, 1), self.vnew.transpose(0, 1)
        a = o.shared_prefix_attention(self.q, self.k, self.v, self.slot_map, self.rows, cu, self.past, None, 128 ** -0.5, self.prefix, causal=True)
        logits = a.float() @ self.head.t()
        accepted, token = o.verify_chains(logits, self.draft, self.drafts, self.cu_drafts, self.accept_u, self.sample_u, temperature=0.8)
        return cu, positions, slots, cu_pages, a, logits, accepted, token


def test_a_serving_step_by_hand():
    s = Step("cpu")
    cu, positions, slots, cu_pages, a, logits, accepted, token = s()
    assert cu.tolist() == [0, 5, 6, 14, 17] and cu_pages.tolist() == [0, 1, 3, 6, 10]
    assert positions.tolist() == [37 + i for i in range(5)] + [53] + [69 + i for i in range(8)] + [85 + i for i in range(3)]
    assert slots.unique().numel() == 17 and torch.equal(slots[:5], s.slot_map[4, 37:42])
    c = dict(q=s.q, k_pool=s.k, v_pool=s.v, slot_map=s.slot_map, seq_rows=s.rows, cu_q=cu, past_lens=s.past, mask_bits=None, scale=128 ** -0.5,
             causal=True)
    attention_close(a, attention_exact(c))
    assert bool((accepted >= 0).all()) and bool((accepted < s.counts).all()) and bool((token >= 0).all())


def same_step(got, want, exact):
    """Integers are equal; ``exact`` is the attention in 64 bits; verification is compared on the same logits."""
    for g, w in zip(got[:4], want[:4]):
        assert g.tolist() == w.tolist()
    attention_close(got[4].cpu(), exact)


@gpu
def test_a_serving_step_with_kernels(clean):
    """Eager, on another stream, and captured: a replay sees what its inputs hold then, and two graphs of one step do not disturb each
    other."""
    cpu, dev = Step("cpu"), Step("cuda")
    want = cpu(ref)

    def exact(s, cu):
        return attention_exact(dict(q=s.q, k_pool=s.k, v_pool=s.v, slot_map=s.slot_map, seq_rows=s.rows, cu_q=cu, past_lens=s.past, mask_bits=None,
                                    scale=128 ** -0.5, causal=True))

    def check(got, s, want, full):
        same_step(got, want, full)
        again = ref.verify_chains(got[5].cpu(), s.draft.cpu(), s.drafts.cpu(), s.cu_drafts.cpu(), s.accept_u.cpu(), s.sample_u.cpu(), temperature=0.8)
        assert got[6].tolist() == again[0].tolist() and got[7].tolist() == again[1].tolist()

    full = exact(cpu, want[0])
    check(dev(), dev, want, full)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dev()
        got2 = dev()
    side.synchronize()
    check(got, dev, want, full)
    check(got2, dev, want, full)

    others = [Step("cuda"), Step("cuda")]
    graphs, outs = [], []
    for s in others:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(s())
    for turn in range(3):
        cpu.counts[:] = torch.tensor([(5, 1, 8, 3), (1, 8, 3, 5), (3, 3, 8, 3)][turn])
        cpu.cu_drafts[1:] = (cpu.counts - 1).cumsum(0)
        cpu.q += 0.25
        for s in others:
            s.counts.copy_(cpu.counts)
            s.cu_drafts.copy_(cpu.cu_drafts)
            s.q.copy_(cpu.q)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want = cpu(ref)
        full = exact(cpu, want[0])
        for s, got in zip(others, outs):
            check(got, s, want, full)


# ------------------------------------------------------------------ in the framework's own paths
def pool_of(device, **kw):
    from jetspec_b200.runtime.kv_pool import PagedKVPool
    return PagedKVPool(1, 1, 8, 10, page_size=4, max_seqs=4, max_seq_len=18, device=device, **kw)


def grow_pools(device):
    from jetspec_b200.runtime.kv_pool import EvictionRequired
    one, many = pool_of(device), pool_of(device)
    asks = [([7, 3, 9], [5, 0, 4]), ([3, 7], [18, 6]), ([7, 7, 9], [9, 13, 4]), ([9], [8]), ([3, 7, 9], [18, 18, 9])]
    for seqs, tokens in asks:
        failed = []
        try:
            for s, n in zip(seqs, tokens):
                one.reserve(s, n)
        except EvictionRequired as e:
            failed.append(str(e))
        try:
            many.reserve_batch(seqs, tokens)
        except EvictionRequired as e:
            failed.append(str(e))
        assert len(failed) in (0, 2) and len(set(failed)) <= 1
        assert torch.equal(one.slot_map, many.slot_map)
        for s in seqs:
            a, b = one.state(s), many.state(s)
            assert (a.row, a.pages, a.capacity) == (b.row, b.pages, b.capacity)
    assert failed and one._refcount == many._refcount and list(one._free_pages) == list(many._free_pages)
    with pytest.raises(EvictionRequired):
        many.reserve_batch([3], [19])
    return many


def causal_rows(pool):
    from jetspec_b200.runtime.attn_metadata import build_attn_metadata
    past, counts = [17, 2, 5], [1, 4, 3]
    m = build_attn_metadata(pool, [3, 9, 7], past, num_query_nodes=counts)
    assert m.cu_q.tolist() == [0, 1, 5, 8] and m.past_lens.tolist() == past and m.seq_rows.tolist() == [pool.state(s).row for s in (3, 9, 7)]
    assert m.positions.tolist() == [17, 2, 3, 4, 5, 5, 6, 7] and (m.max_q, m.num_tokens, m.counts) == (4, 8, counts)
    rows = [pool.slot_map[pool.state(s).row, p:p + n] for s, p, n in zip((3, 9, 7), past, counts)]
    assert torch.equal(m.slots, torch.cat(rows)) and m.causal and m.mask_bits is None
    assert {t.dtype for t in (m.cu_q, m.past_lens, m.seq_rows, m.positions, m.slots)} == {I32}
    two = build_attn_metadata(pool, [9, 9], [1, 4], num_query_nodes=[3, 2])      # neighbouring portions of one sequence
    assert two.positions.tolist() == [1, 2, 3, 4, 5] and torch.equal(two.slots, pool.slot_map[pool.state(9).row, 1:6])


def test_pools_and_batches_plan_their_slots():
    causal_rows(grow_pools("cpu"))


@gpu
def test_pools_and_batches_plan_their_slots_on_the_gpu(clean):
    causal_rows(grow_pools("cuda"))


class Sampler:
    """Draws from the target's logits plus ``noise``."""

    def __init__(self, runner, noise):
        self.runner, self.noise = runner, noise

    def propose_sampled(self, context_ids, k, temperature, target_hidden=None):
        ids, rows = context_ids, []
        for _ in range(k):
            rows.append(self.runner.forward(ids, self.runner.new_cache(64), last_position_logits_only=True)[0][0, -1] + self.noise)
            ids = torch.cat((ids, ops.sample(rows[-1], temperature).view(1, 1)), 1)
        return ids[0, -k:], torch.stack(rows)


def chains_of_a_model(device, monkeypatch):
    from jetspec_b200 import LLM, SamplingParams
    from jetspec_b200.models import Qwen3ForCausalLM, tiny_config
    llm = LLM(Qwen3ForCausalLM.random_init(tiny_config(), seed=0, dtype=torch.float32), device=device, dtype=torch.float32)
    prompt = torch.randint(0, 1024, (1, 9), generator=torch.Generator().manual_seed(0))
    noise = torch.randn(1024, generator=torch.Generator().manual_seed(1)).to(device)
    torch.manual_seed(0)
    calls = []
    monkeypatch.setattr(ops, "verify_chains", lambda *a, _f=ops.verify_chains, **kw: calls.append(kw) or _f(*a, **kw))
    run = lambda shift, t, n: llm.generate_chain(prompt, Sampler(llm.runner, noise * shift), block_size=4, sampling_params=SamplingParams(t, n))
    same = run(0.0, 0.9, 13)                 # drafts from the target's own probabilities are kept, but for rounding
    assert len(same["token_ids"]) == 13 and calls == [dict(temperature=0.9)] * 3
    assert len(run(1.0, 0.9, 10)["token_ids"]) == 10
    # a temperature that counts as none: the target's most likely tokens, whatever was drafted
    want = llm.generate(prompt, SamplingParams(0.0, 12))["token_ids"]
    assert run(3.0, 1e-6, 12)["token_ids"] == want


def test_generate_chain_with_a_sampling_head():
    from jetspec_b200 import LLM, SamplingHeadDrafter, SamplingParams
    from jetspec_b200.models import DraftHeadModel, Qwen3ForCausalLM, draft_head_config, tiny_config
    model = Qwen3ForCausalLM.random_init(tiny_config(), seed=0, dtype=torch.float32)
    head = DraftHeadModel.random_init(draft_head_config(model.config, num_layers=1, block_size=4, num_taps=2), seed=5, dtype=torch.float32)
    drafter = SamplingHeadDrafter(head, model, block_size=4, target_layer_ids=[0, 1])
    llm, prompt = LLM(model, device="cpu", dtype=torch.float32), torch.arange(1, 10).view(1, -1)
    run = lambda t, n: llm.generate_chain(prompt, drafter, block_size=4, target_layer_ids=drafter.target_layer_ids,
                                          sampling_params=SamplingParams(t, n))["token_ids"]
    torch.manual_seed(0)
    assert len(run(1.0, 11)) == 11
    greedy = llm.generate(prompt, SamplingParams(0.0, 11))["token_ids"]
    assert run(1e-6, 11) == greedy and run(0.0, 11) == greedy


def test_generate_chain_verifies_draws(monkeypatch):
    chains_of_a_model("cpu", monkeypatch)


@gpu
def test_generate_chain_verifies_draws_on_the_gpu(clean, monkeypatch):
    chains_of_a_model("cuda", monkeypatch)


