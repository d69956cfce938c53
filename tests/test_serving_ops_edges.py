"""Operators of a batched serving step where they are easily wrong: rows that are not numbers, very large vocabularies and values, views at odd
addresses, padded batches, long items of attention, lengths past the slot map.
"""
import math
import random
import re

import pytest
import torch

from jetspec_b200 import ops
from jetspec_b200.ops import reference as ref
from test_serving_ops import I32, attend, attention_case, attention_close, attention_exact, clean, i32, kernel_refuses  # noqa: F401

gpu = pytest.mark.gpu
INF, NAN = math.inf, math.nan


# ------------------------------------------------------------------ verification of chains
def one_chain(target, draft, x, u, v, dtype=torch.float32, **kw):
    """A chain of one sequence, on the CPU and on the GPU: what the two say."""
    args = [torch.stack(target).to(dtype), torch.stack(draft).to(dtype) if draft else target[0].new_zeros(0, target[0].numel()).to(dtype),
            i32(*x), i32(0, len(x)), torch.tensor(u), torch.tensor([v])]
    got = ops.verify_chains(*[a.cuda() for a in args], **kw)
    return tuple(int(t) for t in ref.verify_chains(*args, **kw)), tuple(int(t) for t in got)


def test_verify_chains_of_rows_that_are_not_numbers():
    """A NaN in a target row: nothing is accepted, no token.  In a draft row: it says nothing, like an empty row."""
    p = torch.tensor([0.5, 0.25, 0.25]).log()
    q = torch.tensor([0.25, 0.5, 0.25]).log()
    bad = torch.tensor([1.0, NAN, 2.0])
    call = lambda target, draft, x, u, v, **kw: tuple(int(t) for t in ops.verify_chains(
        torch.stack(target), torch.stack(draft), i32(*x), i32(0, len(x)), torch.tensor(u), torch.tensor([v]), **kw))
    for kw in (dict(), dict(temperature=0.0)):
        assert call([bad, p], [q], [0], [.0], .5, **kw) == (0, -1)
        assert call([p, bad], [p], [0], [.9], .5, **kw) == (1, -1)
    assert call([p, p], [bad], [2], [.9], .3) == (1, 0)


@gpu
@pytest.mark.parametrize("V,dtype", [(3, torch.float32), (4099, torch.float32), (70001, torch.bfloat16)])
def test_verify_chains_kernel_of_rows_that_are_not_numbers(clean, V, dtype):
    g = torch.Generator().manual_seed(V)
    p, q = (torch.randn(V, generator=g) * 2 for _ in "pq")
    x = int(p.argmax())
    for at in (0, V // 2, V - 1):
        bad, far = p.clone(), p.clone()
        bad[at] = NAN
        far[at] = INF
        for kw in (dict(), dict(temperature=0.0), dict(draft_temperature=0.0), dict(temperature=0.6, draft_temperature=2.0)):
            for target, draft in (([bad, p], [q]), ([p, bad], [p]), ([p, p], [bad]), ([bad, bad], [bad]), ([far, p], [q]), ([p, far], [p]),
                                  ([p, p], [far]), ([far, far], [far])):
                for u in (0.0, 0.9):
                    want, got = one_chain(target, draft, [x], [u], 0.4, dtype, **kw)
                    assert got == want, (at, kw, u)
    # beside sequences whose rows are sound
    target = torch.stack([p, p, bad, p, p]).to(dtype)
    args = [target, torch.stack([p, q]).to(dtype), i32(x, x), i32(0, 1, 2, 2), torch.tensor([.9, .0]), torch.tensor([.3, .6, .8])]
    want, got = ref.verify_chains(*args), ops.verify_chains(*[a.cuda() for a in args])
    assert [t.tolist() for t in got] == [t.tolist() for t in want] and want[0].tolist() == [1, 0, 0] and want[1].tolist()[1] == -1


@gpu
def test_verify_chains_kernel_of_a_vocabulary_of_millions(clean):
    """Sums beyond 2^24 beside masked entries: what is left of ``p - q`` are the two tokens that only the draft masked."""
    V = 2 ** 24 + 19
    target, draft = torch.zeros(2, V, device="cuda"), torch.zeros(1, V, device="cuda")
    target[0, 11], target[0, 12] = -INF, -INF
    draft[0, 5], draft[0, 9] = -INF, -INF
    for v, want in ((0.0, 5), (0.49, 5), (0.51, 9)):
        accepted, token = ops.verify_chains(target, draft, i32(11, device="cuda"), i32(0, 1, device="cuda"), torch.tensor([0.5], device="cuda"),
                                            torch.tensor([v], device="cuda"))
        assert (accepted.tolist(), token.tolist()) == ([0], [want])
    for v in (0.0, 0.25, 0.999):      # behind an accepted draft: the last row, all alike
        accepted, token = ops.verify_chains(target, draft, i32(7, device="cuda"), i32(0, 1, device="cuda"), torch.tensor([0.5], device="cuda"),
                                            torch.tensor([v], device="cuda"))
        v32 = float(torch.tensor(v))
        # the running sum is off by 6e-11 of itself at most, 0.001 of a token here
        assert accepted.tolist() == [1] and abs(int(token) - int(v32 * V)) <= 1


LOWEST = torch.finfo(torch.float32).min


def large_rows(V, g):
    """Rows of values far from zero, and the temperatures at which they say something."""
    flat = lambda v: torch.full((V,), v)
    some = torch.rand(V, generator=g) < 0.3
    some[:2] = torch.tensor([True, False])
    near = flat(2e5)
    near[~some] = float(torch.nextafter(torch.tensor(2e5), torch.tensor(0.0)))
    step = flat(-1e9)
    step[~some] = -1e9 - 64
    usual = torch.randn(V, generator=g) * 3
    return [(flat(-1e9), 0.2), (flat(-1e9), 1.0), (step, 37.0), (flat(-1e30), 1.0), (flat(-1e30).masked_fill(some, -2e30), 0.7),
            (flat(1e30).masked_fill(some, 0.0), 1.0), (flat(LOWEST), 1.0), (flat(LOWEST), 0.01), (flat(LOWEST).masked_fill(some, -INF), 1.0),
            (flat(LOWEST).masked_fill(some, -INF), 1e30), (usual.masked_fill(some, LOWEST), 0.8), (usual.masked_fill(some, -1e9), 0.8),
            (near, 2e-5), (near, 0.01), (usual * 1000, 2e-5), (usual.masked_fill(some, -INF), 1e30), (flat(-LOWEST).masked_fill(some, LOWEST), 0.5),
            (usual * 1e29, 1e29)]


@gpu
@pytest.mark.parametrize("V,dtype", [(1003, torch.float32), (20001, torch.bfloat16)])
def test_verify_chains_kernel_of_large_values(clean, V, dtype):
    """Rows that a finite mask fills, neighbours among large values, temperatures at both ends."""
    g = torch.Generator().manual_seed(V)
    usual = torch.randn(V, generator=g)
    for number, (row, hot) in enumerate(large_rows(V, g)):
        row = row.to(dtype).float()
        if dtype == torch.bfloat16:
            row = row.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)      # the type's own extremes
        x = int(row.argmax())
        for v in (0.0, 0.3, 0.77):
            for kw in (dict(temperature=hot), dict(temperature=torch.tensor([hot]))):
                gpu_kw = lambda d: {k: t.cuda() if torch.is_tensor(t) else t for k, t in d.items()}
                args = [row[None].to(dtype), row[None][:0].to(dtype), i32(), i32(0, 0), torch.zeros(0), torch.tensor([v])]
                assert int(ops.verify_chains(*[a.cuda() for a in args], **gpu_kw(kw))[1]) == int(ref.verify_chains(*args, **kw)[1]), (number, v)
            for u in (0.3, 0.7):
                for target, draft, kw in (([row, row], [row], dict(temperature=hot)), ([usual, row], [row], dict(temperature=1.0, draft_temperature=hot)),
                                          ([row, usual], [usual], dict(temperature=hot, draft_temperature=1.0))):
                    want, got = one_chain(target, draft, [x], [u], v, dtype, **kw)
                    assert got == want, (number, u, v, kw)


def test_verify_chains_refuses_temperatures_without_bounds():
    from jetspec_b200.ops import cuda_ext
    row = torch.zeros(1, 4)
    call = lambda **kw: cuda_ext.verify_chains(row, row[:0], i32(), i32(0, 0), torch.zeros(0), torch.zeros(1), **kw)
    for t in (1.1e30, INF, NAN, -1.0):
        kernel_refuses(lambda: call(temperature=t), "temperature")
        kernel_refuses(lambda: call(draft_temperature=t), "draft_temperature")


def greedy_threshold(device):
    """1e-5 in fp32 lies below 1e-5: the lowest most likely token, although half of the probability is at the next one."""
    row = torch.tensor([[-INF, 0.0, 0.0]], device=device)
    accepted, token = ops.verify_chains(row, row[:0], i32(device=device), i32(0, 0, device=device), torch.zeros(0, device=device),
                                        torch.tensor([0.75], device=device), temperature=torch.tensor([1e-5], device=device))
    assert accepted.tolist() == [0] and token.tolist() == [1]


def test_verify_chains_greedy_threshold():
    greedy_threshold("cpu")


@gpu
def test_verify_chains_kernel_greedy_threshold(clean):
    greedy_threshold("cuda")


@pytest.mark.parametrize("value", [-INF, NAN])
def test_generate_chain_of_a_target_that_says_nothing(monkeypatch, value):
    """Logits without a number among them end the generation with an error, and no -1 is fed to the model."""
    from jetspec_b200 import LLM, SamplingParams
    from jetspec_b200.models import Qwen3ForCausalLM, tiny_config
    llm = LLM(Qwen3ForCausalLM.random_init(tiny_config(), seed=0, dtype=torch.float32), device="cpu", dtype=torch.float32)
    fed, forward = [], llm.runner.forward

    def silent(ids, cache, **kw):
        fed.append(ids)
        logits, cache, hidden = forward(ids, cache, **kw)
        return (logits if len(fed) == 1 else torch.full_like(logits, value)), cache, hidden

    class Drafts:
        def propose_sampled(self, context_ids, k, temperature, target_hidden=None):
            return torch.arange(k), torch.zeros(k, 1024)

    monkeypatch.setattr(llm.runner, "forward", silent)
    torch.manual_seed(0)
    with pytest.raises(RuntimeError, match="logit"):
        llm.generate_chain(torch.arange(1, 8).view(1, -1), Drafts(), block_size=4, sampling_params=SamplingParams(0.8, 20))
    assert len(fed) == 2 and all(int(ids.min()) >= 0 for ids in fed)


@gpu
def test_verify_chains_kernel_cuts_across_a_power_of_two(clean):
    """A maximum just above a negative power of two, at a temperature that sets neighbouring values worlds apart: the values below it, and
    with them what the cut is rounded by, lie twice as far from each other."""
    V, top = 2 ** 24 + 19, -(2.0 ** 14 - 2.0 ** -9)
    assert float(torch.tensor(top)) == top and float(torch.nextafter(torch.tensor(top), torch.tensor(0.0))) == top + 2.0 ** -10
    target, draft = torch.full((2, V), top, device="cuda"), torch.full((1, V), top, device="cuda")
    target[0, 11], target[0, 12] = -INF, -1e5
    draft[0, 5], draft[0, 9] = -INF, -1e5
    for v, want in ((0.0, 5), (0.49, 5), (0.51, 9)):
        accepted, token = ops.verify_chains(target, draft, i32(11, device="cuda"), i32(0, 1, device="cuda"), torch.tensor([0.5], device="cuda"),
                                            torch.tensor([v], device="cuda"), temperature=1e-5)
        assert (accepted.tolist(), token.tolist()) == ([0], [want])


# ------------------------------------------------------------------ attention behind a shared prefix
@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of nothing: not where a mistake would launch a kernel on them")
def test_shared_attention_entry_refuses_addresses():
    """Results leave in stores of 32 bytes, keys and queries come in 16: the entry point turns other addresses down before it starts anything."""
    from jetspec_b200.ops import cuda_ext
    need = cuda_ext.shared_prefix_workspace(1, 2, 2, 1, 64, 0, 2)
    entry = cuda_ext._entry("js_shared_attention", "plppppppppplpiiiiiiiiifiiip")
    sound = dict(q=4096, k=4096, v=4096, out=4096, ws=4096)

    def rc(**kw):
        a = {**sound, **kw}
        return entry(a["q"], 256, a["k"], a["v"], 4096, 4096, 4096, 4096, 0, a["out"], a["ws"], need, 4096, 1, 2, 2, 1, 64, 1, 64, 0, 1, 1.0, 0, 2,
                     cuda_ext.SM_COUNT, None)

    assert rc(out=4096 + 16) == rc(out=4096 + 8) == rc(ws=4096 + 16) == rc(q=4096 + 8) == rc(k=4096 + 8) == rc(v=4096 + 2) == -12


@gpu
def test_shared_prefix_attention_of_views_at_odd_addresses(clean):
    """Queries that start off a 16-byte boundary, one token whose stride says nothing, pools that no copy can read."""
    c = attention_case(3, 8, 2, 70, [0, 9], [2, 3], True, device="cuda")
    want = attention_exact(c)
    flat = torch.zeros(c["q"].numel() + 8, dtype=torch.bfloat16, device="cuda")
    for shift in (1, 4):
        q = flat[shift:shift + c["q"].numel()].view(c["q"].shape)
        q.copy_(c["q"])
        attention_close(attend({**c, "q": q}), want)
    one = attention_case(4, 8, 2, 70, [5], [1], True, device="cuda")
    want = attention_exact(one)
    for stride in (0, 5, 1027, 8 * 128 + 4):
        q = one["q"].as_strided((1, 8, 128), (stride, 128, 1))
        attention_close(attend({**one, "q": q}), want)


def test_shared_prefix_attention_refuses_pools_off_their_boundary():
    from jetspec_b200.ops import cuda_ext
    c = attention_case(0, 4, 2, 20, [0, 5], [4, 3], False)
    for name in ("k_pool", "v_pool"):
        odd = torch.zeros(c[name].numel() + 1, dtype=torch.bfloat16)[1:].view(c[name].shape)
        kernel_refuses(lambda: cuda_ext.shared_prefix_attention(**{**c, "max_q": 4, name: odd}), "16 bytes")


@gpu
def test_shared_prefix_attention_reports_rows_past_the_slot_map(clean):
    """Positions that the slot map has no columns for, and lengths below zero: reported, as slot planning does."""
    for past in (0, 1):                   # with a prefix of its own, and without
        c = attention_case(6, 8, 2, 64 * (1 - past), [0, 7, 0, 3], [1, 1, 1, 1], True, device="cuda")
        most = c["slot_map"].shape[1]
        attend({**c, "past_lens": c["past_lens"] * 0 + most - 1})
        clean.check_status("cuda")
        for lens in ((most, most - 1, most - 1, most - 1), (most - 1, most - 1, most - 1, most + 5), (most - 1, 2 ** 31 - 1, most - 1, most - 1)):
            attend({**c, "past_lens": i32(*lens, device="cuda")})
            with pytest.raises(RuntimeError, match="slot"):
                clean.check_status("cuda")
    c = attention_case(6, 8, 2, 0, [0, 7], [1, 1], True, device="cuda")
    attend({**c, "past_lens": i32(-1, 7, device="cuda")})
    with pytest.raises(RuntimeError, match="slot"):
        clean.check_status("cuda")
    # a sequence without rows has no positions: whatever its length says
    c = attention_case(6, 8, 2, 64, [0, 7, 0], [1, 0, 1], True, device="cuda")
    want = attention_exact(c)
    attention_close(attend({**c, "past_lens": torch.where(i32(0, 1, 0, device="cuda") > 0, 10 ** 6, c["past_lens"]).to(I32)}), want)


@gpu
@pytest.mark.parametrize("idle", [1, 3, 40])
def test_shared_prefix_attention_behind_idle_sequences(clean, idle):
    """A batch whose first sequences have no rows, and slot-map rows that are not theirs any more."""
    c = attention_case(8, 8, 2, 200, [4, 0, 30], [1, 2, 1], True, device="cuda")
    want = attention_exact(c)
    n = c["cu_q"].numel() - 1
    for row in (0, -1, 10 ** 6):          # slots outside the pool, and no row at all
        rows = torch.cat((i32(*[row] * idle, device="cuda"), c["seq_rows"]))
        cu = torch.cat((c["cu_q"].new_zeros(idle), c["cu_q"]))
        past = torch.cat((c["past_lens"].new_zeros(idle), c["past_lens"]))
        assert rows.numel() == n + idle
        attention_close(attend({**c, "seq_rows": rows, "cu_q": cu, "past_lens": past}), want)
        clean.check_status("cuda")


# ------------------------------------------------------------------ slot planning
def padded_plan(device):
    """Requests that fill a batch up: no rows, no pages, any slot-map row.  Nothing about them is wrong."""
    t = lambda *v: i32(*v, device=device)
    slot_map = torch.zeros(3, 32, dtype=I32, device=device)
    cu_q, positions, slots, cu_pages = ops.plan_slots(t(8, 4, 8, 0, 0, 8), t(0, 1, 4, 0, 0, 0), t(2, 1, 2, -1, -1, 1), t(7, 9), 4, slot_map, 7)
    assert cu_q.tolist() == [0, 0, 1, 5, 5, 5, 5] and cu_pages.tolist() == [0, 0, 1, 2, 2, 2, 2]
    assert positions.tolist() == [4, 8, 9, 10, 11, 0, 0] and slots.tolist() == [28, 36, 37, 38, 39, -1, -1]


def test_plan_slots_of_a_padded_batch():
    padded_plan("cpu")


@gpu
def test_plan_slots_kernel_of_a_padded_batch(clean):
    padded_plan("cuda")
    clean.check_status("cuda")
    ops.plan_slots(i32(4, 4, device="cuda"), i32(0, 4, device="cuda"), i32(9, 9, device="cuda"), i32(1, 2, device="cuda"), 4,
                   torch.zeros(3, 32, dtype=I32, device="cuda"), 4, mapped_lens=i32(4, 8, device="cuda"))
    with pytest.raises(RuntimeError, match="status 5"):      # rows there are, and their request's slot-map row is not
        clean.check_status("cuda")
    ops.plan_slots(i32(4, device="cuda"), i32(0, device="cuda"), i32(9, device="cuda"), i32(1, 2, device="cuda"), 4,
                   torch.zeros(3, 32, dtype=I32, device="cuda"), 0, mapped_lens=i32(0, device="cuda"))
    with pytest.raises(RuntimeError, match="status 5"):      # a page was granted, and its slots have nowhere to go
        clean.check_status("cuda")


# ------------------------------------------------------------------ attention when a wait has run out: that cannot be staged on a GPU
def shared_attention_source():
    from jetspec_b200.ops import cuda_ext
    source = next(s for s in cuda_ext.sources() if s.endswith("attn_shared_sm100.cu"))
    return re.sub(r"//.*", "", open(source).read())


def test_shared_attention_merge_stays_in_its_workspace():
    """The merge finds a sequence's parts by where the plan says that its item begins, which a CTA whose wait ran out has not written.  Its
    expressions, on any number: the CTAs are some that there are.  On places of a line as the plan has them, the bounds change nothing."""
    text = shared_attention_source()
    own = re.search(r"const int u = own_begin = (.*);\s*c0 = (.*);\s*own = (.*);", text).groups()
    python = [re.sub(r"(?<!/)/(?!/)", "//", re.sub(r"p\.plan\[1 \+ item\]", "said", e)).replace("p.ctas", "ctas") for e in own]

    def parts(said, piece, units, two, ctas=148, cost=8):
        env = dict(said=said, piece=piece, units=units, two=two, ctas=ctas, kItemCost=cost, min=min, max=max)
        for name, expression in zip(("u", "c0", "own"), python):
            env[name] = eval(expression, env)
            assert -2 ** 31 <= env[name] < 2 ** 31
        return env["u"], env["c0"], env["own"]

    rng = random.Random(0)
    for _ in range(2000):
        piece, units, two = rng.choice([1, 7, 900, 13_000_000]), rng.randint(1, 2000), rng.randint(0, 1)
        u, c0, own = parts(rng.choice([-2 ** 31, -1, 2 ** 31 - 1, rng.randint(-2 ** 31, 2 ** 31 - 1)]), piece, units, two)
        assert 0 <= c0 < 148 and 1 <= own <= 148 - c0
        length = (units << two) + 8
        if length <= 148 * piece:
            begin = rng.randint(0, 148 * piece - length)
            u, c0, own = parts(begin, piece, units, two)
            assert (u, c0, own) == (begin, (begin + 8) // piece, (begin + 8 + ((units - 1) << two)) // piece - (begin + 8) // piece + 1)


def test_shared_attention_settles_what_it_started():
    """A role whose wait runs out leaves its loop with copies or products in flight.  Every ring that a warp starts something on is waited for
    behind the loops, use by use, ahead of the barrier that the CTA's tensor memory is given back behind."""
    text = shared_attention_source()
    body = re.search(r"void sa_settle\(.*?\n}", text, re.S).group()
    assert "int j = max(0, uses - SLOTS); j < uses; ++j" in body and "mbar_wait(&ring[j % SLOTS], (j / SLOTS) & 1," in body
    loaders, scores, outputs, softmax = re.split(r"\} else if \(warp == 8\) \{|\} else if \(warp == 11\) \{|\n  \} else \{\n",
                                                 text[text.index("if (warp == 9 || warp == 10)"):text.index("attn_shared_merge_kernel")])[:4]
    settled = lambda role: re.findall(r"sa_settle<(.*?), p\.status", role)
    assert settled(loaders) == ["KSLOTS>(values ? kv_full + KSLOTS : kv_full, n", "2>(q_full, uses"]
    assert settled(scores) == ["2>(s_full, n"] and settled(outputs) == ["2>(pv_done, n"]
    end = softmax[softmax.rindex("sa_tmem_st_wait()"):]
    assert "tcgen05" not in end and end.index("__syncthreads()") < end.index("tmem_dealloc")
    for role, commits in ((scores, "umma_commit(&s_full[g])"), (outputs, "umma_commit(&pv_done[g])")):      # a commit of that ring for every use
        assert role.count(commits) == 1 and "++job, ++n" in role


# ------------------------------------------------------------------ attention: many items a CTA, many sequences
def line_of_work(c):
    """Restated from the kernel's description: the segments of every CTA on the line of items, as (units of the segment, units of the item,
    both tiles of the pair have rows, of the prefix)."""
    keys, cost, ctas = 96, 8, 148
    T, hq, _ = c["q"].shape
    hkv = c["k_pool"].shape[0]
    npt = 128 // (hq // hkv)
    cu, past = c["cu_q"].tolist(), c["past_lens"].tolist()
    B = len(past)
    shared = 4 * T <= 3 * max(B * npt, T + B * npt // 2)
    prefix = c["prefix_len"] // 16 * 16 if shared else 0
    seqs = ([(cu[-1], prefix, prefix, 0, True)] if prefix else []) + [(cu[b + 1] - cu[b], past[b], past[b] + cu[b + 1] - cu[b], prefix, False)
                                                                      for b in range(B)]
    items = []
    for n, committed, end, first, common in seqs:
        for pair in range(-(-n // (2 * npt))):
            last = min(end, committed + (pair + 1) * 2 * npt) if c["causal"] and not common else end
            units, two = -(-max(0, last - first) // keys), n - pair * 2 * npt > npt
            items += [(units, two, common)] * (hkv * (units > 0))
    total = sum((u << two) + cost for u, two, _ in items)
    piece = max(1, -(-total // ctas))
    segments, at = [[] for _ in range(ctas)], 0
    begins = lambda t, two: (max(0, t - cost) + two) >> two
    for units, two, common in items:
        length = (units << two) + cost
        for cta in range(at // piece, (at + length - 1) // piece + 1):
            lo, hi = max(at, cta * piece) - at, min(at + length, (cta + 1) * piece) - at
            part = begins(hi, two) - begins(lo, two)
            if part > 0:
                segments[cta].append((part, units, two, common))
        at += length
    return segments


LONG = dict(heads=64, kv_heads=16, prefix=600, behind=[(37 * i) % 400 for i in range(16)], counts=[64 + (29 * i) % 65 for i in range(16)])
MANY = [(500, 40, 4), (769, 16, 2)]


@pytest.mark.parametrize("causal", [False, True])
def test_long_items_come_whole(causal):
    """What the test on the GPU below is about: CTAs with several items that they finish alone, of several units, beside items that are cut."""
    segments = line_of_work(attention_case(7, causal=causal, **LONG))
    whole = [[s for s in cta if s[0] == s[1] and s[2]] for cta in segments]
    assert sum(len(w) >= 2 and min(s[1] for s in w) >= 7 for w in whole) >= 20 and not any(s[3] for cta in segments for s in cta)
    assert sum(s[0] < s[1] for cta in segments for s in cta) >= 50


@gpu
@pytest.mark.parametrize("causal", [False, True])
def test_shared_prefix_attention_of_long_items(clean, causal):
    c = attention_case(7, causal=causal, device="cuda", **LONG)
    want = attention_exact(c)
    got = attend(c, max_q=128)
    attention_close(got, want)
    assert torch.equal(got, attend(c, max_q=128))


@gpu
@pytest.mark.parametrize("B,heads,kv", MANY)
def test_shared_prefix_attention_of_many_sequences(clean, B, heads, kv):
    """More sequences than a CTA has threads: their lengths are summed in rounds."""
    c = attention_case(B, heads, kv, 150, [(13 * i) % 60 for i in range(B)], [1 + (i % 7 == 3) for i in range(B)], True, device="cuda", slack=1.0)
    want = attention_exact(c)
    attention_close(attend(c, max_q=2), want)
    attention_close(attend({**c, "prefix_len": 0}, max_q=2), want)
