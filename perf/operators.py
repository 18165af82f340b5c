"""The operators around a paged 8-bit cache, as cases that can be timed: rotary
positions, the append (with the rotation in the same call), attention from
single tokens to whole prompts, and the calls that share, reserve and compact
pages.

`own` false computes each in plain torch, `own` true calls the library.

The cache: pools [n_pages][block_tokens][num_kv][head_dim] of e4m3 codes and one
power-of-two exponent (a byte, biased by 127) for each page and KV head.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a decode step of eight slots: q and k inside one projection buffer, a quarter of each head rotated
        dict(name="rope_step", kind="rope", tokens=8, num_q=16, num_kv=4, hd=256, rot=64, layout="half",
             scaling="none", inverse=False, far=40000),
        # a long prompt in one call, whole heads, adjacent pairs, positions stretched to a million
        dict(name="rope_prompt", kind="rope", tokens=32768, num_q=24, num_kv=4, hd=128, rot=128,
             layout="interleaved", scaling="yarn", inverse=False, far=1000000),
        # a decode step of 32 slots: q and k rotated and the new rows appended, most into pages begun earlier
        dict(name="append_step", kind="append", slots=32, tok_lo=1, tok_hi=1, ctx_lo=100, ctx_hi=16000, num_q=16,
             num_kv=4, hd=256, bt=64, rot=64, layout="half", lens=11),
        # two prompts' rows, already rotated, quantized into their pages
        dict(name="append_prompt", kind="append", slots=2, tok_lo=9000, tok_hi=16384, ctx_lo=1, ctx_hi=300, num_q=24,
             num_kv=4, hd=256, bt=64, rot=0, layout="half", lens=12),
        # a chat's first answers: one slot, a few hundred keys, where latency is all there is
        dict(name="step_short", kind="attn", slots=1, tok_lo=1, tok_hi=1, ctx_lo=701, ctx_hi=701, num_q=16, num_kv=4,
             hd=256, bt=64, window=0, sink=0, lens=1),
        # one long conversation's decode step
        dict(name="step_128k", kind="attn", slots=1, tok_lo=1, tok_hi=1, ctx_lo=131071, ctx_hi=131071, num_q=16,
             num_kv=4, hd=256, bt=256, window=0, sink=0, lens=2),
        # continuous batching: 32 slots of ragged lengths in small pages, GQA 6
        dict(name="step_32slots", kind="attn", slots=32, tok_lo=1, tok_hi=1, ctx_lo=500, ctx_hi=32768, num_q=24,
             num_kv=4, hd=128, bt=16, window=0, sink=0, lens=3),
        # speculative blocks of up to 12 tokens in four slots at 32K..64K keys
        dict(name="verify_4slots", kind="attn", slots=4, tok_lo=5, tok_hi=12, ctx_lo=32768, ctx_hi=65536, num_q=16,
             num_kv=4, hd=256, bt=64, window=0, sink=0, lens=4),
        # a long prompt's later chunk
        dict(name="chunk_32k", kind="attn", slots=1, tok_lo=2048, tok_hi=2048, ctx_lo=32000, ctx_hi=32000, num_q=16,
             num_kv=4, hd=256, bt=64, window=0, sink=0, lens=5),
        # several new prompts of odd lengths at once, a sliding window with sinks
        dict(name="prompts_ragged", kind="attn", slots=6, tok_lo=150, tok_hi=4000, ctx_lo=0, ctx_hi=0, num_q=32,
             num_kv=4, hd=128, bt=32, window=1500, sink=16, lens=6),
        # parallel samples: prompts forked to children, every slot's next page made its own
        dict(name="fork_step", kind="fork", slots=8, children=3, ctx_lo=500, ctx_hi=8000, layers=4, num_kv=4, hd=256,
             bt=64, spare=200, lens=7),
        # a pool two thirds empty after its long slots ended, pushed together
        dict(name="compact_pool", kind="compact", slots=48, ctx_lo=500, ctx_hi=16000, layers=2, num_kv=4, hd=256,
             bt=64, keep=0.35, lens=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "step", "step", "verify", "chunk", "chunk", "fork", "compact"])
    nq, kv = rng.choice([(16, 4), (16, 4), (24, 4), (32, 4), (8, 8)])
    hd = rng.choice([128, 256])
    bt = rng.choice([16, 32, 64, 64, 256])
    lens = rng.randint(100, 10 ** 6)
    if kind == "rope":
        rot = rng.choice([hd, hd // 2, hd // 4, 2 * rng.randint(5, hd // 2)])
        return dict(kind=kind, tokens=_log(rng, 1, 16384), num_q=nq, num_kv=kv, hd=hd, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    inverse=rng.random() < 0.4, far=_log(rng, 1000, 1000000))
    if kind == "append":
        long = rng.random() < 0.5
        hi = _log(rng, 200, 8000) if long else rng.randint(1, 9)
        return dict(kind=kind, slots=rng.randint(1, 3) if long else _log(rng, 1, 64), tok_lo=max(1, hi // 3), tok_hi=hi,
                    ctx_lo=1, ctx_hi=_log(rng, 10, 8000), num_q=nq, num_kv=kv, hd=hd, bt=bt,
                    rot=rng.choice([0, hd, hd // 4]), layout=rng.choice(["half", "interleaved"]), lens=lens)
    if kind == "fork":
        return dict(kind=kind, slots=rng.randint(1, 12), children=rng.randint(1, 4), ctx_lo=100, ctx_hi=_log(rng, 200, 8000),
                    layers=rng.randint(1, 4), num_kv=kv, hd=hd, bt=bt, spare=rng.randint(100, 400), lens=lens)
    if kind == "compact":
        return dict(kind=kind, slots=rng.randint(4, 48), ctx_lo=200, ctx_hi=_log(rng, 400, 12000), layers=rng.randint(1, 2),
                    num_kv=4, hd=hd, bt=rng.choice([32, 64, 256]), keep=round(rng.uniform(0.2, 0.8), 2), lens=lens)
    c = dict(kind="attn", num_q=nq, num_kv=kv, hd=hd, bt=bt, window=0, sink=0, lens=lens)
    if kind == "step":
        slots = _log(rng, 1, 48)
        hi = _log(rng, 200, 131072 // max(1, slots // 4))
        c.update(slots=slots, tok_lo=1, tok_hi=1, ctx_lo=max(1, hi // rng.randint(1, 16)), ctx_hi=hi)
    elif kind == "verify":
        hi = _log(rng, 200, 32768)
        c.update(slots=rng.randint(1, 6), tok_lo=2, tok_hi=rng.randint(3, 16), ctx_lo=max(1, hi // 4), ctx_hi=hi)
    else:
        hi = _log(rng, 40, 2048)
        c.update(slots=rng.randint(1, 4), tok_lo=max(1, hi // rng.randint(1, 20)), tok_hi=hi, ctx_lo=0,
                 ctx_hi=rng.choice([0, _log(rng, 100, 8000)]))
    if rng.random() < 0.3:
        c.update(window=_log(rng, 64, 8192), sink=rng.choice([0, rng.randint(1, 100)]))
    return c


def _lens(case):
    """New tokens and earlier keys of every slot."""
    r = random.Random(case["lens"])
    between = lambda lo, hi: _log(r, lo, hi) if lo > 0 else r.randint(lo, hi)  # noqa: E731
    n = [between(case.get("tok_lo", 1), case.get("tok_hi", 1)) for _ in range(case["slots"])]
    return n, [between(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["slots"])]


def _seen(p, window, sink):
    """How many keys the query at position p sees."""
    if window <= 0 or p < window:
        return p + 1
    return window + min(sink, p - window + 1)


def work(case):
    kind, hd = case["kind"], case.get("hd", 0)
    if kind == "rope":
        rows = case["tokens"] * (case["num_q"] + case["num_kv"])
        return {"bytes": 4 * rows * case["rot"], "flops": 3 * rows * case["rot"]}
    if kind in ("fork", "compact"):
        page = case["layers"] * 2 * case["num_kv"] * (case["bt"] * hd + 1)
        _, ctx = _lens(case)
        bt = case["bt"]
        if kind == "fork":
            entries = case["children"] * sum(-(-c // bt) for c in ctx)
            copies = (1 + case["children"]) * sum(c % bt > 0 for c in ctx)
            return {"bytes": 2 * copies * page + 16 * entries, "flops": 0}
        _, ref, moves = _compact_layout(case)
        return {"bytes": 2 * moves * page + 8 * len(ref) + 8 * case["slots"] * _max_blocks(case), "flops": 0}
    n, ctx = _lens(case)
    kv = case["num_kv"] * hd
    if kind == "append":
        total = sum(n)
        byts = 2 * total * kv * 3
        if case["rot"]:
            byts += total * case["num_q"] * hd * 4
        return {"bytes": byts, "flops": 4 * total * kv}
    w, s = case["window"], case["sink"]
    pairs = sum(_seen(c + t, w, s) for k, c in zip(n, ctx) for t in range(k))
    keys = sum(_seen(c + k - 1, w + k - 1 if w > 0 else 0, s) for k, c in zip(n, ctx))
    return {"bytes": 2 * keys * kv + 4 * sum(n) * case["num_q"] * hd, "flops": 4 * hd * case["num_q"] * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _rows(g, *shape):
    """fp16 rows of N(0, 1) with 2% of the channels eight times as large."""
    x = torch.randn(*shape, device=DEV, generator=g)
    loud = torch.rand(shape[-2:], device=DEV, generator=g) < 0.02
    return (x * (1.0 + 7.0 * loud)).half()


def _pow2(n):
    """2^n exactly, fp32 (n an integer tensor, -126..127)."""
    return ((n.int() + 127) << 23).view(torch.float32)


def _exponent(amax):
    """Smallest biased exponent e >= 95 with amax <= 448 * 2^(e - 127) (amax fp32 or wider)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e, -32).clamp_min(-32) + 127


def _codes(x, e):
    """fp32 x over 2^(e - 127), to e4m3 codes (bytes)."""
    return (x * _pow2(127 - e)).to(torch.float8_e4m3fn).view(torch.uint8)


def _filled_pool(g, n_pages, bt, kv, hd):
    x = _rows(g, n_pages, bt, kv, hd).float()
    e = _exponent(x.abs().amax((1, 3)))
    return _codes(x, e[:, None, :, None]), e.to(torch.uint8)


def _max_blocks(case):
    n, ctx = _lens(case)
    return max(-(-(a + b) // case["bt"]) for a, b in zip(n, ctx)) + 1


def _paged(case, g):
    """Shuffled pages for every slot's tokens; tables, positions and starts."""
    n, ctx = _lens(case)
    bt, mb = case["bt"], _max_blocks(case)
    need = [-(-(a + b) // bt) for a, b in zip(n, ctx)]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, device=DEV, generator=g).int()
    tables = torch.full((case["slots"], mb), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, k in enumerate(need):
        tables[s, :k] = order[at:at + k]
        at += k
    kp, ke = _filled_pool(g, n_pages, bt, case["num_kv"], case["hd"])
    vp, ve = _filled_pool(g, n_pages, bt, case["num_kv"], case["hd"])
    starts = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=DEV)
    return dict(kp=kp, ke=ke, vp=vp, ve=ve, tables=tables, starts=starts,
                positions=torch.tensor(ctx, dtype=torch.int32, device=DEV), total=sum(n), max_tok=max(n),
                max_ctx=max(a + b for a, b in zip(n, ctx)))


def _scaling(case):
    return {"none": None, "linear": ("linear", 4.0), "ntk": ("ntk", 4.0),
            "yarn": ("yarn", 8.0, 32768)}[case.get("scaling", "none")]


def _frequencies(rot, scaling):
    """Radians a position, in 64 bits, and the amplitude."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    base, amp = 10000.0, 1.0
    if scaling and scaling[0] == "ntk":
        base *= scaling[1] ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if scaling and scaling[0] == "linear":
        f = f / scaling[1]
    if scaling and scaling[0] == "yarn":
        keep = ((scaling[2] * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f, amp = keep * f + (1 - keep) * f / scaling[1], 1.0 + 0.1 * math.log(scaling[1])
    return f.to(DEV), amp


def _pool_state(case, g, n_pages):
    """Layers of pools filled with bytes, as the page calls see them."""
    shape = (case["layers"], n_pages, case["bt"], case["num_kv"], case["hd"])
    pools = torch.randint(0, 120, (2,) + shape, dtype=torch.uint8, device=DEV, generator=g)
    exps = torch.randint(95, 136, (2,) + shape[:2] + (case["num_kv"],), dtype=torch.uint8, device=DEV, generator=g)
    return pools, exps


def _compact_layout(case):
    """Tables, reference counts and the number of pages to move: slots placed in random pages, then some ended."""
    r = random.Random(case["lens"] + 1)
    _, ctx = _lens(case)
    need = [-(-c // case["bt"]) for c in ctx]
    n_pages = sum(need) + 64
    order = list(range(n_pages))
    r.shuffle(order)
    mb = _max_blocks(case)
    tables, ref, at = np.full((case["slots"], mb), -1, np.int32), np.zeros(n_pages, np.int32), 0
    alive = [r.random() < case["keep"] for _ in need]
    alive[0] = True
    for s, k in enumerate(need):
        if alive[s]:
            tables[s, :k] = order[at:at + k]
            ref[order[at:at + k]] = 1
        at += k
    used = int((ref > 0).sum())
    return tables, ref, int((ref[used:] > 0).sum())


def prepare(case, seed):
    g = _gen(seed, 7)
    kind = case["kind"]
    st = {"case": case}
    if kind in ("rope", "append"):
        nq, kv, hd = case["num_q"], case["num_kv"], case["hd"]
        if kind == "append":
            st.update(_paged(case, g))
        tokens = case.get("tokens") or st["total"]
        # one projection's output: q, k and v of a token side by side
        qkv = torch.cat([_rows(g, tokens, nq, hd), _rows(g, tokens, kv, hd), _rows(g, tokens, kv, hd)], 1)
        st.update(q=qkv[:, :nq], k=qkv[:, nq:nq + kv], v=qkv[:, nq + kv:])
        if kind == "rope":
            st["positions"] = torch.randint(0, case["far"], (tokens,), dtype=torch.int32, device=DEV, generator=g)
            st["k_out"] = torch.empty_like(st["k"], memory_format=torch.contiguous_format)
        st["q_out"] = torch.empty(tokens, nq, hd, dtype=torch.float16, device=DEV)
        if case["rot"]:
            st["freq"], st["amp"] = _frequencies(case["rot"], _scaling(case))
            if own:
                from qengine_amd import kvcache
                st["rope"] = kvcache.rope_table(case["rot"], base=10000.0, scaling=_scaling(case), device=DEV)
    elif kind == "attn":
        st.update(_paged(case, g))
        # three rows behind the last slot's, as a padded batch has
        st["q"] = torch.randn(st["total"] + 3, case["num_q"], case["hd"], device=DEV, generator=g).half()
        st["out"] = torch.zeros_like(st["q"])
        if own:
            from qengine_amd import kvcache
            st["ws"] = kvcache.attn_f8_paged_workspace(case["num_q"], case["num_kv"], case["slots"], st["total"] + 3,
                                                       st["max_tok"], st["max_ctx"], DEV, head_dim=case["hd"])
    elif kind == "fork":
        _, ctx = _lens(case)
        bt, mb = case["bt"], _max_blocks(case)
        need = [-(-c // bt) for c in ctx]
        n_pages = sum(need) + case["spare"]
        pools, exps = _pool_state(case, g, n_pages)
        order = torch.randperm(n_pages, device=DEV, generator=g).int()
        total = case["slots"] * (1 + case["children"])
        tables = torch.full((total, mb), -1, dtype=torch.int32, device=DEV)
        at = 0
        for s, k in enumerate(need):
            tables[s, :k] = order[at:at + k]
            at += k
        ref = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
        ref[order[:at].long()] = 1
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        kids = list(range(case["slots"], total))
        par = [(k - case["slots"]) % case["slots"] for k in kids]
        st.update(pools=pools, exps=exps, tables=tables, ref=ref, parents=i32(par), children=i32(kids),
                  fork_tokens=i32([ctx[p] for p in par]), none=i32([0] * len(kids)), slots=i32(list(range(total))),
                  positions=i32(ctx + [ctx[p] for p in par]), one=i32([1] * total), status=i32([0] * total))
    else:
        tables, ref, _ = _compact_layout(case)
        pools, exps = _pool_state(case, g, len(ref))
        meta = torch.from_numpy(np.concatenate([tables.reshape(-1), ref])).to(DEV)
        st.update(pools=pools, exps=exps, meta0=meta, meta=meta.clone(), shape=tables.shape,
                  moved=torch.empty(len(ref), dtype=torch.int32, device=DEV),
                  n_used=torch.zeros(1, dtype=torch.int32, device=DEV))
    if kind in ("fork", "compact") and own:
        from qengine_amd import kvcache
        st["planes"] = kvcache.page_planes([t[i, j] for t in (st["pools"], st["exps"]) for i in range(2)
                                            for j in range(case["layers"])])
    return st


# ---------------------------------------------------------------------------
# one pass: the library's calls
# ---------------------------------------------------------------------------

def _own_run(st):
    from qengine_amd import kvcache
    c = st["case"]
    kind = c["kind"]
    if kind == "rope":
        kvcache.rope(st["q"], st["k"], st["positions"], st["rope"], layout=c["layout"], inverse=c["inverse"],
                     q_out=st["q_out"], k_out=st["k_out"])
        return {"q": st["q_out"], "k": st["k_out"]}
    if kind == "append":
        more = dict(q=st["q"], q_out=st["q_out"], rope=st["rope"], layout=c["layout"]) if c["rot"] else {}
        kvcache.f8_append_kv_paged(st["k"], st["v"], st["kp"], st["vp"], st["ke"], st["ve"], st["tables"],
                                   st["starts"], st["positions"], max_tok=st["max_tok"], **more)
        return _append_out(st)
    if kind == "attn":
        kvcache.attn_f8_paged(st["q"], st["kp"], st["vp"], st["ke"], st["ve"], st["out"], st["ws"], st["tables"],
                              st["starts"], st["positions"], max_tok=st["max_tok"], max_ctx=st["max_ctx"],
                              scale=1.0 / math.sqrt(c["hd"]), window=c["window"], sink=c["sink"])
        return st["out"]
    if kind == "fork":
        kvcache.pages_release(st["tables"], st["ref"], st["children"], st["none"], block_tokens=c["bt"])
        kvcache.pages_fork(st["tables"], st["ref"], st["parents"], st["children"], st["fork_tokens"], st["status"],
                           block_tokens=c["bt"])
        kvcache.pages_reserve(st["tables"], st["ref"], st["slots"], st["positions"], st["one"], st["status"],
                              st["planes"], block_tokens=c["bt"], max_new=1)
        return _fork_out(st)
    st["meta"].copy_(st["meta0"])
    tables, ref = _compact_views(st)
    kvcache.pages_compact(tables, ref, st["moved"], st["n_used"], st["planes"])
    return {"meta": st["meta"], "n_used": st["n_used"], "pools": st["pools"], "exps": st["exps"]}


def _append_out(st):
    out = {"k": st["kp"].view(torch.float8_e4m3fn), "v": st["vp"].view(torch.float8_e4m3fn), "ke": st["ke"],
           "ve": st["ve"]}
    return {**out, "q": st["q_out"]} if st["case"]["rot"] else out


def _fork_out(st):
    return {"tables": st["tables"], "ref": st["ref"], "status": st["status"], "pools": st["pools"], "exps": st["exps"]}


def _compact_views(st):
    slots, mb = st["shape"]
    return st["meta"][:slots * mb].view(slots, mb), st["meta"][slots * mb:]


# ---------------------------------------------------------------------------
# one pass: plain torch
# ---------------------------------------------------------------------------

def _rotate(x, positions, freq, amp, layout, inverse):
    """fp16 x [tokens][heads][hd], angles in 64 bits and products in 32."""
    a = positions.double()[:, None] * freq
    cos, sin = (a.cos() * amp).float()[:, None], (a.sin() * (-amp if inverse else amp)).float()[:, None]
    r = 2 * freq.numel()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if layout == "interleaved" else (y[..., :r // 2], y[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if layout == "interleaved" else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., r:]], -1).half()


def _token_index(st):
    """Slot and position of every packed token."""
    t = torch.arange(st["total"], device=DEV, dtype=torch.int32)
    slot = torch.bucketize(t, st["starts"][1:], right=True)
    return slot, st["positions"][slot] + t - st["starts"][slot]


def _append_plain(st, x, pool, exps, slot, pos):
    bt = st["case"]["bt"]
    x = torch.nan_to_num(x, nan=0.0).clamp(-61440, 61440).float()
    page = st["tables"][slot, pos // bt].long()
    top = torch.zeros_like(exps, dtype=torch.float32)
    top.scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
    new = _exponent(top)
    # the page that a slot's first new token continues keeps its older rows
    off = st["positions"] % bt
    first = st["tables"].gather(1, (st["positions"] // bt).long()[:, None])[:, 0].long()
    was = exps[first].int()
    e = torch.where((off > 0)[:, None], torch.maximum(new[first], was), new[first])
    new[first] = e
    old = pool[first]
    again = _codes(old.view(torch.float8_e4m3fn).float(), (e - was + 127)[:, None, :, None])
    older = torch.arange(bt, device=DEV) < off[:, None]
    pool[first] = torch.where(older[:, :, None, None], again, old)
    touched = torch.unique(page)
    exps[touched] = new[touched].to(torch.uint8)
    pool[page, (pos % bt).long()] = _codes(x, new[page][..., None])


def _visible(pos, keys, window, sink):
    seen = keys <= pos
    if window > 0:
        seen = seen & ((keys > pos - window) | (keys < sink))
    return seen


def _attn_plain(st):
    c = st["case"]
    bt, nq, kv, hd = c["bt"], c["num_q"], c["num_kv"], c["hd"]
    slots, width, g = c["slots"], st["max_tok"], nq // kv
    keys = torch.arange(st["max_ctx"], device=DEV)
    page = st["tables"][:, keys // bt].long()
    there = page >= 0
    page = page.clamp_min(0)

    def rows(pool, exps):   # [slots][kv][keys][hd]
        x = pool[page, keys % bt].view(torch.float8_e4m3fn).float()
        return (x * _pow2(exps[page].int() - 127)[..., None]).permute(0, 2, 1, 3).contiguous()

    n = (st["starts"][1:] - st["starts"][:-1]).long()
    t = torch.arange(width, device=DEV)
    at = (st["starts"][:-1, None] + t).clamp_max(st["total"] - 1).long()          # [slots][width]
    q = st["q"][at].float().view(slots, width, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(slots, kv, width * g, hd)
    s = torch.matmul(q, rows(st["kp"], st["ke"]).transpose(2, 3)).view(slots, kv, width, g, -1) / math.sqrt(hd)
    pos = st["positions"][:, None] + t
    seen = _visible(pos[..., None], keys, c["window"], c["sink"]) & there[:, None]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = torch.matmul(p.view(slots, kv, width * g, -1), rows(st["vp"], st["ve"])).view(slots, kv, width, g, hd)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(slots, width, nq, hd)
    live = t < n[:, None]
    st["out"][at[live]] = o[live].half()
    return st["out"]


def _release_plain(tables, ref, slots, keep, bt):
    rows = tables[slots.long()]
    gone = (rows >= 0) & (torch.arange(rows.shape[1], device=DEV) >= ((keep + bt - 1) // bt)[:, None])
    ref -= torch.bincount(rows[gone], minlength=ref.numel()).int()
    tables[slots.long()] = torch.where(gone, -1, rows)


def _fork_plain(tables, ref, parents, children, tokens, status, bt):
    rows = tables[parents.long()]
    kept = torch.arange(rows.shape[1], device=DEV) < ((tokens + bt - 1) // bt)[:, None]
    ref += torch.bincount(rows[kept], minlength=ref.numel()).int()
    tables[children.long()] = torch.where(kept, rows, -1)
    status[:children.numel()] = 0


def _reserve_plain(st):
    """One new token a slot: at most one page of each is asked for."""
    tables, ref, bt = st["tables"], st["ref"], st["case"]["bt"]
    slots, block = st["slots"].long(), (st["positions"] // bt).long()
    page = tables[slots, block]
    shared = (page >= 0) & (ref[page.clamp_min(0).long()] > 1)
    want = (page < 0) | shared
    free = (ref == 0).nonzero()[:, 0]
    rank = torch.cumsum(want.int(), 0)
    served = rank <= free.numel()
    st["status"].copy_(torch.where(served, 0, -9))
    take, shared = want & served, shared & served
    fresh = free[(rank - 1).clamp(0, max(0, free.numel() - 1))]
    copy = shared & (st["positions"] % bt > 0)
    src, dst = page[copy].long(), fresh[copy]
    st["pools"][:, :, dst] = st["pools"][:, :, src]
    st["exps"][:, :, dst] = st["exps"][:, :, src]
    ref -= torch.bincount(page[shared], minlength=ref.numel()).int()
    ref[fresh[take]] = 1
    tables[slots[take], block[take]] = fresh[take].int()


def _compact_plain(st):
    st["meta"].copy_(st["meta0"])
    tables, ref = _compact_views(st)
    used = ref > 0
    n = used.sum()
    at = torch.arange(ref.numel(), device=DEV)
    src, dst = (used & (at >= n)).nonzero()[:, 0], (~used & (at < n)).nonzero()[:, 0]
    to = at.int()
    to[src] = dst.int()
    st["pools"][:, :, dst] = st["pools"][:, :, src]
    st["exps"][:, :, dst] = st["exps"][:, :, src]
    tables.copy_(torch.where(tables >= 0, to[tables.clamp_min(0).long()], tables))
    ref[dst] = ref[src]
    ref[src] = 0
    st["n_used"][0] = n
    return {"meta": st["meta"], "n_used": st["n_used"], "pools": st["pools"], "exps": st["exps"]}


def _plain_run(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "rope":
        st["q_out"].copy_(_rotate(st["q"], st["positions"], st["freq"], st["amp"], c["layout"], c["inverse"]))
        st["k_out"].copy_(_rotate(st["k"], st["positions"], st["freq"], st["amp"], c["layout"], c["inverse"]))
        return {"q": st["q_out"], "k": st["k_out"]}
    if kind == "append":
        slot, pos = _token_index(st)
        k = st["k"]
        if c["rot"]:
            k = _rotate(k, pos, st["freq"], st["amp"], c["layout"], False)
            st["q_out"].copy_(_rotate(st["q"], pos, st["freq"], st["amp"], c["layout"], False))
        _append_plain(st, k, st["kp"], st["ke"], slot, pos)
        _append_plain(st, st["v"], st["vp"], st["ve"], slot, pos)
        return _append_out(st)
    if kind == "attn":
        return _attn_plain(st)
    if kind == "fork":
        bt = c["bt"]
        _release_plain(st["tables"], st["ref"], st["children"], st["none"], bt)
        _fork_plain(st["tables"], st["ref"], st["parents"], st["children"], st["fork_tokens"], st["status"], bt)
        _reserve_plain(st)
        return _fork_out(st)
    return _compact_plain(st)


def run(state):
    if own:
        return _own_run(state)
    else:
        return _plain_run(state)


# ---------------------------------------------------------------------------
# 64-bit results from the definitions
# ---------------------------------------------------------------------------

def _turn64(x, positions, case):
    """x [tokens][heads][hd] in 64 bits, each pair times e^(i theta) as a complex number."""
    f, amp = _frequencies(case["rot"], _scaling(case))
    r = case["rot"]
    theta = positions.double()[:, None, None] * f * (-1.0 if case.get("inverse") else 1.0)
    y = x.double().clone()
    if case["layout"] == "half":
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous())
        z = z * torch.polar(torch.full_like(theta, amp), theta)
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous())
        y[..., :r] = torch.view_as_real(z * torch.polar(torch.full_like(theta, amp), theta)).flatten(-2)
    return y


def _grid64(x):
    """Nearest e4m3 values (ties to even) of 64-bit x within +-448."""
    _, e = torch.frexp(x)
    step = _pow2((e - 4).clamp_min(-9)).double()
    return torch.round(x / step) * step


def _append64(st, x, pool, exps):
    bt = st["case"]["bt"]
    out = pool.view(torch.float8_e4m3fn).double()
    starts, first = st["starts"].tolist(), st["positions"].tolist()
    tables = st["tables"].tolist()
    for s, p0 in enumerate(first):
        t, end = starts[s], starts[s + 1]
        while t < end:
            p = p0 + t - starts[s]
            k = min(end - t, bt - p % bt)
            page, row = tables[s][p // bt], p % bt
            new = x[t:t + k].clamp(-61440, 61440)
            e = torch.ceil(torch.log2(new.abs().amax((0, 2)).clamp_min(2.0 ** -40) / 448)).clamp_min(-32)
            if row:
                was = exps[page].double() - 127
                e = torch.maximum(e, was)
                out[page, :row] = _grid64(out[page, :row] * _pow2(was - e)[:, None])
            out[page, row:row + k] = _grid64(new * _pow2(-e)[:, None])
            t += k
    return out


def _attn64(st):
    c = st["case"]
    bt, nq, kv, hd = c["bt"], c["num_q"], c["num_kv"], c["hd"]
    g = nq // kv
    out = st["out"].double()
    starts, first = st["starts"].tolist(), st["positions"].tolist()
    for s, p0 in enumerate(first):
        t0, t1 = starts[s], starts[s + 1]
        length = p0 + t1 - t0
        j = torch.arange(length, device=DEV)
        page = st["tables"][s].long()[j // bt]
        for h in range(kv):
            k, v = (pool[page, j % bt, h].view(torch.float8_e4m3fn).double() * _pow2(ex[page, h].int() - 127)[:, None]
                    for pool, ex in ((st["kp"], st["ke"]), (st["vp"], st["ve"])))
            for a in range(t0, t1, 512):
                b = min(t1, a + 512)
                pos = p0 + torch.arange(a - t0, b - t0, device=DEV)
                hide = j > pos[:, None]
                if c["window"] > 0:
                    hide |= (j <= pos[:, None] - c["window"]) & (j >= c["sink"])
                x = st["q"][a:b, h * g:(h + 1) * g].double().reshape(-1, hd) @ k.T.contiguous() / math.sqrt(hd)
                x = x.view(b - a, g, length).masked_fill(hide[:, None], -math.inf).softmax(-1)
                out[a:b, h * g:(h + 1) * g] = (x.view(-1, length) @ v).view(b - a, g, hd)
    return out


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None   # whole numbers
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return {n: _turn64(st[n], st["positions"], case) for n in ("q", "k")}
    if case["kind"] == "attn":
        return _attn64(st)
    slot, pos = _token_index(st)
    k = st["k"].double()
    if case["rot"]:
        k = _turn64(st["k"], pos, case).half().double()   # the rows are fp16 before they are quantized
    out = {"k": _append64(st, k, st["kp"], st["ke"]), "v": _append64(st, st["v"].double(), st["vp"], st["ve"]),
           "ke": None, "ve": None}
    return {**out, "q": _turn64(st["q"], pos, case)} if case["rot"] else out
