"""The operators of a decoding loop over a paged 8-bit cache, as cases that can be timed: norms of
query and key heads with the rotation (and their gradient), attention weight accumulated for each key,
eviction of the keys with the least of it, beam search's selection, and the reordering of slots that
follows it.

`own` false computes each in plain torch, `own` true calls the library.

The cache: pools [n_pages][block_tokens][num_kv][head_dim] of e4m3 codes, one power-of-two exponent (a
byte, biased by 127) for each page and KV head, and accumulated weights [n_pages][num_kv][block_tokens].
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
        # a decode step of eight slots: q and k inside one projection buffer, a quarter of each head turned
        dict(name="norm_step", kind="norm", tokens=8, num_q=16, num_kv=4, hd=256, rot=64, layout="half",
             scaling="none", far=40000),
        # a long prompt in one call, whole heads, adjacent pairs, positions stretched to a million
        dict(name="norm_prompt", kind="norm", tokens=32768, num_q=32, num_kv=4, hd=128, rot=128,
             layout="interleaved", scaling="yarn", far=1000000),
        # a training step's rows: gradients of the heads and of both weights
        dict(name="norm_grad", kind="grad", tokens=8192, num_q=16, num_kv=4, hd=256, rot=64, layout="half",
             scaling="none", far=8192),
        # a decode step of 32 slots adds its queries' weights to those of all keys so far
        dict(name="weigh_step", kind="weigh", slots=32, tok_lo=1, tok_hi=1, ctx_lo=500, ctx_hi=32768, num_q=16,
             num_kv=4, hd=256, bt=64, window=0, sink=0, decay=1.0, fresh=False, lens=3),
        # after long prompts: their last 64 queries weigh every key, before a first eviction
        dict(name="weigh_window", kind="weigh", slots=4, tok_lo=64, tok_hi=64, ctx_lo=8000, ctx_hi=32768, num_q=32,
             num_kv=4, hd=128, bt=64, window=0, sink=0, decay=1.0, fresh=True, lens=4),
        # two whole prompts of odd lengths: every query weighs the keys before it
        dict(name="weigh_prompt", kind="weigh", slots=2, tok_lo=1500, tok_hi=4000, ctx_lo=0, ctx_hi=0, num_q=16,
             num_kv=4, hd=256, bt=32, window=0, sink=0, decay=0.9, fresh=False, lens=5),
        # one long conversation cut to an eighth
        dict(name="evict_long", kind="evict", slots=1, ctx_lo=131072, ctx_hi=131072, part=0.125, num_kv=4, hd=256,
             bt=256, sink=4, recent=64, lens=6),
        # continuous batching in small pages: every slot gives back 15% of its keys
        dict(name="evict_batch", kind="evict", slots=24, ctx_lo=1500, ctx_hi=9000, part=0.85, num_kv=8, hd=128, bt=16,
             sink=16, recent=128, lens=7),
        # one request's beam step in fp32
        dict(name="beam_one", kind="beam", n=1, beams=4, vocab=32003, take=8, dtype="float32", first=False, lens=8),
        # a batch of beam searches over a large vocabulary
        dict(name="beam_batch", kind="beam", n=64, beams=8, vocab=131072, take=16, dtype="float16", first=False, lens=9),
        # the slots of one request's beams take over their parents' pages and token histories
        dict(name="reorder_one", kind="reorder", n=1, beams=4, ctx_lo=700, ctx_hi=2000, bt=64, history=2048, state=0,
             lens=10),
        # the same for 64 requests, with a per-slot state beside the pages
        dict(name="reorder_batch", kind="reorder", n=64, beams=8, ctx_lo=500, ctx_hi=16000, bt=64, history=16384,
             state=262144, lens=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "grad", "step", "step", "window", "prompt", "evict", "evict", "beam", "beam", "reorder"])
    nq, kv = rng.choice([(16, 4), (16, 4), (32, 4), (20, 4), (8, 8)])
    hd = rng.choice([128, 256])
    bt = rng.choice([16, 32, 64, 64, 256])
    lens = rng.randint(100, 10 ** 6)
    if kind in ("norm", "grad"):
        hd = rng.choice([64, 128, 128, 256, 256, 80, 2 * rng.randint(20, 150)])
        rot = rng.choice([hd, hd // 4 * 2, 2 * rng.randint(5, hd // 2), 0])
        return dict(kind=kind, tokens=_log(rng, 1, 16384 if kind == "norm" else 6000), num_q=nq, num_kv=kv, hd=hd, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    far=_log(rng, 1000, 1000000))
    if kind == "evict":
        slots = _log(rng, 1, 32)
        hi = _log(rng, 200, 131072 // slots)
        return dict(kind=kind, slots=slots, ctx_lo=max(1, hi // rng.randint(1, 12)), ctx_hi=hi,
                    part=round(rng.uniform(0.05, 0.99), 3), num_kv=kv, hd=hd, bt=bt, sink=rng.randint(0, 40),
                    recent=rng.choice([0, rng.randint(1, 300)]), lens=lens)
    if kind == "beam":
        beams = rng.randint(1, 12)
        return dict(kind=kind, n=_log(rng, 1, 48), beams=beams, vocab=_log(rng, 900, 131072),
                    take=rng.choice([beams, 2 * beams]), dtype=rng.choice(["float16", "bfloat16", "float32"]),
                    first=rng.random() < 0.2, lens=lens)
    if kind == "reorder":
        return dict(kind=kind, n=_log(rng, 1, 64), beams=rng.randint(2, 8), ctx_lo=100, ctx_hi=_log(rng, 200, 16000), bt=bt,
                    history=_log(rng, 64, 8192), state=rng.choice([0, 16 * _log(rng, 1, 8192)]), lens=lens)
    c = dict(kind="weigh", num_q=nq, num_kv=kv, hd=hd, bt=bt, window=0, sink=0, decay=rng.choice([1.0, 0.95, 0.0]),
             fresh=rng.random() < 0.3, lens=lens)
    if kind == "step":
        slots = _log(rng, 1, 40)
        hi = _log(rng, 200, 131072 // max(1, slots // 4))
        c.update(slots=slots, tok_lo=1, tok_hi=rng.choice([1, 1, 3]), ctx_lo=max(1, hi // rng.randint(1, 16)), ctx_hi=hi)
    elif kind == "window":
        hi = _log(rng, 100, 24000)
        c.update(slots=rng.randint(1, 4), tok_lo=8, tok_hi=rng.randint(9, 64), ctx_lo=max(1, hi // 3), ctx_hi=hi)
    else:
        hi = _log(rng, 40, 2500)
        c.update(slots=rng.randint(1, 3), tok_lo=max(1, hi // rng.randint(1, 9)), tok_hi=hi, ctx_lo=0,
                 ctx_hi=rng.choice([0, _log(rng, 100, 2000)]))
    if rng.random() < 0.3:
        c.update(window=_log(rng, 64, 8192), sink=rng.choice([0, rng.randint(1, 100)]))
    return c


def _lens(case):
    """New tokens and earlier keys of every slot."""
    r = random.Random(case["lens"])
    between = lambda lo, hi: _log(r, lo, hi) if lo > 0 else r.randint(lo, hi)  # noqa: E731
    n = [between(case.get("tok_lo", 1), case.get("tok_hi", 1)) for _ in range(case["slots"])]
    return n, [between(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["slots"])]


def _beam_lens(case):
    """Tokens of every request's beams."""
    r = random.Random(case["lens"])
    return [_log(r, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["n"])]


def _kept(case):
    """Rows that every slot keeps."""
    return [max(1, int(c * case["part"])) for c in _lens(case)[1]]


def _seen(p, window, sink):
    """How many keys the query at position p sees."""
    if window <= 0 or p < window:
        return p + 1
    return window + min(sink, p - window + 1)


def work(case):
    kind = case["kind"]
    if kind in ("norm", "grad"):
        x = case["tokens"] * (case["num_q"] + case["num_kv"]) * case["hd"]
        return {"bytes": (4 if kind == "norm" else 6) * x, "flops": (7 if kind == "norm" else 14) * x}
    if kind == "beam":
        x = case["n"] * case["beams"] * case["vocab"]
        return {"bytes": x * (4 if case["dtype"] == "float32" else 2), "flops": 4 * x}
    if kind == "reorder":
        slots = case["n"] * case["beams"]
        entries = case["beams"] * sum(-(-c // case["bt"]) for c in _beam_lens(case))
        return {"bytes": 8 * entries + 2 * slots * (4 * case["history"] + case["state"]), "flops": 0}
    n, ctx = _lens(case)
    kv, hd = case["num_kv"], case["hd"]
    if kind == "evict":
        moved = sum(max(0, k - case["sink"]) for k in _kept(case))
        return {"bytes": kv * (4 * sum(ctx) + moved * (4 * hd + 8)), "flops": 0}
    w, s = case["window"], case["sink"]
    pairs = sum(_seen(c + t, w, s) for k, c in zip(n, ctx) for t in range(k))
    keys = sum(_seen(c + k - 1, w + k - 1 if w > 0 else 0, s) for k, c in zip(n, ctx))
    weights = kv * 4 * (sum(c + k for k, c in zip(n, ctx)) + (0 if case["fresh"] else sum(ctx)))
    return {"bytes": keys * kv * hd + 2 * sum(n) * case["num_q"] * hd + weights, "flops": 2 * hd * case["num_q"] * pairs}


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


def _filled_pool(g, n_pages, bt, kv, hd):
    """Codes and exponents of random rows, each exponent the smallest that holds its page's."""
    x = _rows(g, n_pages, bt, kv, hd).float()
    m, e = torch.frexp(x.abs().amax((1, 3)))
    e = e - 9 + (m > 0.875).int()
    return ((x * _pow2(-e)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8),
            (e + 127).to(torch.uint8))


def _max_blocks(case):
    n, ctx = _lens(case)
    return max(-(-(a + b) // case["bt"]) for a, b in zip(n, ctx)) + 1


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _paged(case, g):
    """Shuffled pages for every slot's tokens, and the weights of their keys so far."""
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
    # a few keys have most of the weight, many next to none
    weights = torch.rand(n_pages, case["num_kv"], bt, device=DEV, generator=g) ** 8
    return dict(kp=kp, ke=ke, weights=weights, tables=tables, n=n, ctx=ctx)


def _scaling(case):
    return {"none": None, "linear": ("linear", 4.0), "ntk": ("ntk", 4.0),
            "yarn": ("yarn", 8.0, 32768)}[case["scaling"]]


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


def _prepare_norm(case, g):
    nq, kv, hd, tokens = case["num_q"], case["num_kv"], case["hd"], case["tokens"]
    # one projection's output: q, k and v of a token side by side
    qkv = torch.cat([_rows(g, tokens, nq, hd), _rows(g, tokens, kv, hd), _rows(g, tokens, kv, hd)], 1)
    st = dict(q=qkv[:, :nq], k=qkv[:, nq:nq + kv],
              positions=torch.randint(0, case["far"], (tokens,), dtype=torch.int32, device=DEV, generator=g),
              wq=1.0 + 0.3 * torch.randn(hd, device=DEV, generator=g), wk=1.0 + 0.3 * torch.randn(hd, device=DEV, generator=g),
              q_out=torch.empty(tokens, nq, hd, dtype=torch.float16, device=DEV),
              k_out=torch.empty(tokens, kv, hd, dtype=torch.float16, device=DEV))
    if case["kind"] == "grad":
        st.update(dq=torch.randn(tokens, nq, hd, device=DEV, generator=g).half(),
                  dk=torch.randn(tokens, kv, hd, device=DEV, generator=g).half(),
                  dwq=torch.empty(hd, device=DEV), dwk=torch.empty(hd, device=DEV))
    st["freq"], st["amp"] = _frequencies(case["rot"], _scaling(case) if case["rot"] else None)
    if own:
        from qengine_amd import kvcache
        st["rope"] = kvcache.rope_table(case["rot"], base=10000.0, scaling=_scaling(case), device=DEV) if case["rot"] else None
        if case["kind"] == "grad":
            st["ws"] = kvcache.norm_rope_grad_workspace(tokens, nq, kv, hd, DEV)
    return st


def _prepare_weigh(case, g):
    st = _paged(case, g)
    n, ctx = st["n"], st["ctx"]
    # three rows behind the last slot's, as a padded batch has
    rows = sum(n) + 3
    st.update(q=torch.randn(rows, case["num_q"], case["hd"], device=DEV, generator=g).half(),
              starts=_i32(np.cumsum([0] + n)), positions=_i32(ctx), total=sum(n), max_tok=max(n),
              max_ctx=max(a + b for a, b in zip(n, ctx)), weighed=_i32([0] * len(n) if case["fresh"] else ctx))
    if own:
        from qengine_amd import kvcache
        st["ws"] = kvcache.weigh_f8_paged_workspace(case["num_q"], case["num_kv"], case["slots"], rows, st["max_tok"],
                                                    st["max_ctx"], DEV, head_dim=case["hd"])
    return st


def _prepare_evict(case, g):
    st = _paged(case, g)
    st["vp"], st["ve"] = _filled_pool(g, st["kp"].shape[0], case["bt"], case["num_kv"], case["hd"])
    keep = _kept(case)
    st.update(lens=_i32(st["ctx"]), keep=_i32(keep), max_ctx=max(st["ctx"]), max_keep=max(keep),
              kept=torch.empty(case["slots"], case["num_kv"], max(keep), dtype=torch.int32, device=DEV))
    if own:
        from qengine_amd import kvcache
        st["ws"] = kvcache.evict_f8_paged_workspace(case["slots"], case["num_kv"], case["bt"], st["max_ctx"], st["max_keep"], DEV)
    return st


def _prepare_beam(case, g):
    n, beams, vocab, take = case["n"], case["beams"], case["vocab"], case["take"]
    x = 2.5 * torch.randn(n * beams, vocab, device=DEV, generator=g)
    # a few likely tokens a row, and forbidden ones
    x.scatter_add_(1, torch.randint(0, vocab, (n * beams, 6), device=DEV, generator=g),
                   12.0 * torch.rand(n * beams, 6, device=DEV, generator=g))
    x.masked_fill_(torch.rand(n * beams, vocab, device=DEV, generator=g) < 0.01, -math.inf)
    scores = (-40.0 * torch.rand(n, beams, device=DEV, generator=g)).sort(1, descending=True).values
    if case["first"]:
        scores[:, 1:] = -math.inf   # (all beams of a request are the same before the first step)
    done = (torch.rand(n, beams, device=DEV, generator=g) < (0.0 if case["first"] else 0.1)).int()
    st = dict(logits=x.to(getattr(torch, case["dtype"])), scores=scores, done=done,
              parents=torch.empty(n, take, dtype=torch.int32, device=DEV),
              tokens=torch.empty(n, take, dtype=torch.int32, device=DEV), top=torch.empty(n, take, device=DEV))
    if own:
        from qengine_amd import kvcache
        st["ws"] = kvcache.beam_select_workspace(n, beams, vocab, take, DEV)
    return st


def _prepare_reorder(case, g):
    n, beams, bt = case["n"], case["beams"], case["bt"]
    lens = [c for c in _beam_lens(case) for _ in range(beams)]
    mb = max(-(-c // bt) for c in lens) + 1
    # a request's beams share their first half and have the rest for themselves
    tables, at = np.full((n * beams, mb), -1, np.int32), 0
    for s, c in enumerate(lens):
        nb = -(-c // bt)
        half = 0 if s % beams == 0 else nb // 2
        tables[s, :half] = tables[s - s % beams, :half]
        tables[s, half:nb] = np.arange(at, at + nb - half)
        at += nb - half
    order = torch.randperm(at + 8, device=DEV, generator=g).int()
    tables = torch.from_numpy(tables).to(DEV)
    tables = torch.where(tables >= 0, order[tables.clamp_min(0).long()], -1).int()
    ref = torch.bincount(tables[tables >= 0].long(), minlength=at + 8).int()
    slots = torch.arange(n * beams, dtype=torch.int32, device=DEV)
    parents = slots // beams * beams + torch.randint(0, beams, (n * beams,), device=DEV, generator=g).int()
    st = dict(tables=tables, ref=ref, slots=slots, parents=parents, n_tokens=_i32(lens),
              status=torch.zeros(n * beams, dtype=torch.int32, device=DEV),
              history=torch.randint(0, 32000, (n * beams, case["history"]), dtype=torch.int32, device=DEV, generator=g),
              state=torch.randint(0, 255, (n * beams, case["state"]), dtype=torch.uint8, device=DEV, generator=g))
    if own:
        from qengine_amd import kvcache
        st["planes"] = kvcache.page_planes([st["history"]] + ([st["state"]] if case["state"] else []))
    return st


_PREPARE = {"norm": _prepare_norm, "grad": _prepare_norm, "weigh": _prepare_weigh, "evict": _prepare_evict,
            "beam": _prepare_beam, "reorder": _prepare_reorder}


def prepare(case, seed):
    return {"case": case, **_PREPARE[case["kind"]](case, _gen(seed, 7))}


# ---------------------------------------------------------------------------
# one pass: the library's calls
# ---------------------------------------------------------------------------

def _own_run(st):
    from qengine_amd import kvcache
    c = st["case"]
    kind = c["kind"]
    if kind == "norm":
        kvcache.norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["positions"], st["rope"], eps=1e-6, layout=c["layout"],
                          q_out=st["q_out"], k_out=st["k_out"])
    elif kind == "grad":
        kvcache.norm_rope_grad(st["q"], st["k"], st["dq"], st["dk"], st["wq"], st["wk"], st["positions"], st["rope"],
                               st["dwq"], st["dwk"], eps=1e-6, layout=c["layout"], q_grad=st["q_out"], k_grad=st["k_out"],
                               workspace=st["ws"])
    elif kind == "weigh":
        kvcache.weigh_f8_paged(st["q"], st["kp"], st["ke"], st["weights"], st["ws"], st["tables"], st["starts"],
                               st["positions"], max_tok=st["max_tok"], max_ctx=st["max_ctx"], scale=1.0 / math.sqrt(c["hd"]),
                               decay=c["decay"], weighed=st["weighed"], window=c["window"], sink=c["sink"])
    elif kind == "evict":
        kvcache.evict_f8_paged(st["kp"], st["vp"], st["ke"], st["ve"], st["weights"], st["tables"], st["lens"], st["keep"],
                               st["kept"], st["ws"], max_ctx=st["max_ctx"], sink=c["sink"], recent=c["recent"])
    elif kind == "beam":
        kvcache.beam_select(st["logits"], st["scores"], st["parents"], st["tokens"], st["top"], st["ws"], done=st["done"],
                            end_token=2)
    else:
        kvcache.pages_reorder(st["tables"], st["ref"], st["slots"], st["parents"], st["n_tokens"], st["status"],
                              st["planes"], block_tokens=c["bt"])


def _outputs(st):
    kind = st["case"]["kind"]
    if kind == "norm":
        return {"q": st["q_out"], "k": st["k_out"]}
    if kind == "grad":
        return {"q": st["q_out"], "k": st["k_out"], "wq": st["dwq"], "wk": st["dwk"]}
    if kind == "weigh":
        return st["weights"]
    if kind == "evict":
        return {"k": st["kp"].view(torch.float8_e4m3fn), "v": st["vp"].view(torch.float8_e4m3fn), "ke": st["ke"],
                "ve": st["ve"], "weights": st["weights"], "kept": st["kept"]}
    if kind == "beam":
        return {"parents": st["parents"], "tokens": st["tokens"], "scores": st["top"]}
    return {"tables": st["tables"], "ref": st["ref"], "status": st["status"], "history": st["history"], "state": st["state"]}


# ---------------------------------------------------------------------------
# one pass: plain torch
# ---------------------------------------------------------------------------

def _pairs(x, rot, layout):
    """The two members of every turned pair, and the rest."""
    if layout == "interleaved":
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]


def _turn(x, st, inverse):
    """fp32 x [tokens][heads][hd], angles in 64 bits."""
    c = st["case"]
    a = st["positions"].double()[:, None] * st["freq"]
    amp = st["amp"]
    cos, sin = (a.cos() * amp).float()[:, None], (a.sin() * (-amp if inverse else amp)).float()[:, None]
    p, q, rest = _pairs(x, c["rot"], c["layout"])
    p, q = p * cos - q * sin, p * sin + q * cos
    turned = torch.stack([p, q], -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat([p, q], -1)
    return torch.cat([turned, rest], -1)


def _norm_plain(st, x, w):
    y = x.float()
    return _turn(y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w, st, False).half()


def _grad_plain(st, x, dy, w):
    y = x.float()
    r = torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    y = y * r
    g = _turn(dy.float(), st, True)
    h = g * w
    dw = (g * y).double().sum((0, 1)).float()
    return (r * (h - y * (h * y).mean(-1, keepdim=True))).half(), dw


def _visible(pos, keys, window, sink):
    seen = keys <= pos
    if window > 0:
        seen = seen & ((keys > pos - window) | (keys < sink))
    return seen


def _weigh_plain(st):
    c = st["case"]
    bt, nq, kv, hd = c["bt"], c["num_q"], c["num_kv"], c["hd"]
    slots, width, g = c["slots"], st["max_tok"], nq // kv
    keys = torch.arange(st["max_ctx"], device=DEV)
    page = st["tables"][:, keys // bt].long().clamp_min(0)
    k = st["kp"][page, keys % bt].view(torch.float8_e4m3fn).float()
    k = (k * _pow2(st["ke"][page].int() - 127)[..., None]).permute(0, 2, 3, 1).contiguous()
    n = (st["starts"][1:] - st["starts"][:-1]).long()
    t = torch.arange(width, device=DEV)
    at = (st["starts"][:-1, None] + t).clamp_max(st["total"] - 1).long()          # [slots][width]
    q = st["q"][at].float().view(slots, width, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(slots, kv, width * g, hd)
    s = torch.matmul(q, k).view(slots, kv, width, g, -1).mul_(1.0 / math.sqrt(hd))
    seen = _visible((st["positions"][:, None] + t)[..., None], keys, c["window"], c["sink"]) & (t < n[:, None])[..., None]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    s.mul_(1.0 / s.sum(-1, keepdim=True).clamp_min(1e-30))
    added = s.sum((2, 3)).permute(0, 2, 1)                                         # [slots][keys][kv]
    there = keys < (st["positions"] + n)[:, None]
    old = st["weights"][page, :, keys % bt]
    new = torch.where((keys < st["weighed"][:, None])[..., None], c["decay"] * old, 0.0) + added
    row = (keys % bt).expand(slots, -1)[there]
    st["weights"][page[there], :, row] = new[there]


def _evict_plain(st):
    c = st["case"]
    bt, kv, slots, hd = c["bt"], c["num_kv"], c["slots"], c["hd"]
    lens, keep, mk = st["lens"].long(), st["keep"].long(), st["max_keep"]
    rows = torch.arange(st["max_ctx"], device=DEV)
    page = st["tables"][:, rows // bt].long().clamp_min(0)
    w = st["weights"][page, :, rows % bt].permute(0, 2, 1)                         # [slots][kv][rows]
    # rows kept whatever their weight are above all others, rows that do not exist below
    own_n = keep.clamp_max(c["recent"])
    first = (keep - own_n).clamp_max(c["sink"])
    always = (rows >= (lens - own_n)[:, None]) | (rows < first[:, None])
    w_key = torch.where(always[:, None], math.inf, w).masked_fill_((rows >= lens[:, None])[:, None], -math.inf)
    # stable: of equal weights the lower row first
    order = w_key.sort(stable=True, dim=-1, descending=True).indices[..., :mk]
    live = torch.arange(mk, device=DEV) < keep[:, None]                            # [slots][mk]
    kept = torch.where(live[:, None], order, 1 << 30).sort(-1).values
    st["kept"].copy_(torch.where(live[:, None], kept, -1))
    src = kept.clamp_max(st["max_ctx"] - 1)
    to = torch.arange(mk, device=DEV)
    nb = -(-mk // bt)
    head = torch.arange(kv, device=DEV)[None, :, None]
    from_page = page.gather(1, src.flatten(1)).view_as(src)
    to_page = page[:, :mk]
    ws = st["weights"][from_page, head, src % bt]
    at = live.nonzero(as_tuple=True)
    into = to_page[at], (to % bt).expand(slots, -1)[at]
    st["weights"][into[0], :, into[1]] = ws.permute(0, 2, 1)[at]
    for pool, exps in ((st["kp"], st["ke"]), (st["vp"], st["ve"])):
        x = pool[from_page, src % bt, head]                                        # [slots][kv][mk][hd]
        e = exps[from_page, head].int().masked_fill(~live[:, None], 0)
        top = torch.nn.functional.pad(e, (0, nb * bt - mk)).view(slots, kv, nb, bt).amax(-1)
        new = top.repeat_interleave(bt, -1)[..., :mk]
        codes = (x.view(torch.float8_e4m3fn).float() * _pow2((e - new).clamp_min(-126))[..., None]).to(torch.float8_e4m3fn)
        pool[into] = codes.view(torch.uint8).permute(0, 2, 1, 3)[at]
        b = (torch.arange(nb, device=DEV) < ((keep + bt - 1) // bt)[:, None]).nonzero(as_tuple=True)
        exps[st["tables"][:, :nb].long()[b]] = top.permute(0, 2, 1)[b].to(torch.uint8)


def _beam_plain(st):
    c = st["case"]
    n, beams, vocab, take = c["n"], c["beams"], c["vocab"], c["take"]
    x = st["logits"].float().nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(-3.4e38)
    total = (x - m).double().exp().sum(-1)
    # of each beam the largest, ties to the lower token: one whole number orders both
    bits = x.add_(0.0).view(torch.int32)
    bits = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(vocab, device=DEV))
    token = torch.topk(key, min(take, vocab), -1).indices.sort(-1).values           # [n * beams][take]
    score = st["scores"].view(-1, 1).double() + (x.gather(1, token).double() - m.double() - total.log()[:, None])
    done = st["done"].view(-1, 1) != 0
    alone = torch.where(torch.arange(token.shape[1], device=DEV) == 0, st["scores"].view(-1, 1).double(), -math.inf)
    token, score = torch.where(done, 2, token).view(n, -1), torch.where(done, alone, score).view(n, -1)
    score = score.nan_to_num(nan=-math.inf, neginf=-math.inf)
    best, order = score.sort(stable=True, dim=-1, descending=True)
    k = min(take, order.shape[1])
    best, order = best[:, :k], order[:, :k]
    there = best > -math.inf
    parent = torch.arange(n, device=DEV)[:, None] * beams + order // (score.shape[1] // beams)
    st["parents"].fill_(-1)[:, :k] = torch.where(there, parent, -1).int()
    st["tokens"].fill_(-1)[:, :k] = torch.where(there, token.gather(1, order), -1).int()
    st["top"].fill_(-math.inf)[:, :k] = best.float()


def _reorder_plain(st):
    tables, ref, bt = st["tables"], st["ref"], st["case"]["bt"]
    slots, parents = st["slots"].long(), st["parents"].long()
    old, rows = tables[slots], tables[parents]
    rows = torch.where(torch.arange(tables.shape[1], device=DEV) < ((st["n_tokens"] + bt - 1) // bt)[:, None], rows, -1)
    size = ref.numel()
    ref += torch.bincount(rows.flatten().long() + 1, minlength=size + 1)[1:].int()
    ref -= torch.bincount(old.flatten().long() + 1, minlength=size + 1)[1:].int()
    tables[slots] = rows
    st["history"][slots] = st["history"][parents]
    st["state"][slots] = st["state"][parents]
    st["status"].zero_()


def _plain_run(st):
    kind = st["case"]["kind"]
    if kind == "norm":
        st["q_out"].copy_(_norm_plain(st, st["q"], st["wq"]))
        st["k_out"].copy_(_norm_plain(st, st["k"], st["wk"]))
    elif kind == "grad":
        dx, dw = _grad_plain(st, st["q"], st["dq"], st["wq"])
        st["q_out"].copy_(dx)
        st["dwq"].copy_(dw)
        dx, dw = _grad_plain(st, st["k"], st["dk"], st["wk"])
        st["k_out"].copy_(dx)
        st["dwk"].copy_(dw)
    else:
        {"weigh": _weigh_plain, "evict": _evict_plain, "beam": _beam_plain, "reorder": _reorder_plain}[kind](st)


def run(state):
    if own:
        _own_run(state)
    else:
        _plain_run(state)
    return _outputs(state)


# ---------------------------------------------------------------------------
# 64-bit results from the definitions
# ---------------------------------------------------------------------------

def _turn64(x, positions, case, sign):
    """x [tokens][heads][hd] in 64 bits, each pair times e^(i theta) as a complex number."""
    if not case["rot"]:
        return x
    f, amp = _frequencies(case["rot"], _scaling(case))
    r = case["rot"]
    theta = positions.double()[:, None, None] * f * sign
    by = torch.polar(torch.full_like(theta, amp), theta)
    y = x.clone()
    if case["layout"] == "half":
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * by
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous()) * by
        y[..., :r] = torch.view_as_real(z).flatten(-2)
    return y


def _norm64(st, x, w, dy=None):
    """Rows, or the gradients of rows and weight for those of the rows' outputs."""
    x, w = x.double(), w.double()
    length = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
    scale = (length ** 2 / x.shape[-1] + 1e-6) ** -0.5
    if dy is None:
        return _turn64(x * scale * w, st["positions"], st["case"], 1.0)
    g = _turn64(dy.double(), st["positions"], st["case"], -1.0)
    inner = torch.einsum("thd,thd,d->th", g, x, w)[..., None]
    return scale * g * w - scale ** 3 / x.shape[-1] * inner * x, torch.einsum("thd,thd,th->d", g, x, scale[..., 0])


def _keys64(pool, exps, page, row, h):
    return pool[page, row, h].view(torch.float8_e4m3fn).double() * _pow2(exps[page, h].int() - 127).double()[:, None]


def _weigh64(st):
    c = st["case"]
    bt, nq, kv, hd = c["bt"], c["num_q"], c["num_kv"], c["hd"]
    g = nq // kv
    out = st["weights"].double()
    starts, first, old = st["starts"].tolist(), st["positions"].tolist(), st["weighed"].tolist()
    for s, p0 in enumerate(first):
        t0, t1 = starts[s], starts[s + 1]
        length = p0 + t1 - t0
        j = torch.arange(length, device=DEV)
        page = st["tables"][s].long()[j // bt]
        for h in range(kv):
            k = _keys64(st["kp"], st["ke"], page, j % bt, h)
            added = torch.zeros(length, dtype=torch.float64, device=DEV)
            for a in range(t0, t1, 256):
                b = min(t1, a + 256)
                pos = p0 + torch.arange(a - t0, b - t0, device=DEV)
                hide = j > pos[:, None]
                if c["window"] > 0:
                    hide |= (j <= pos[:, None] - c["window"]) & (j >= c["sink"])
                x = st["q"][a:b, h * g:(h + 1) * g].double().reshape(-1, hd) @ k.T.contiguous() / math.sqrt(hd)
                added += x.view(b - a, g, length).masked_fill(hide[:, None], -math.inf).softmax(-1).sum((0, 1))
            was = out[page, h, j % bt] * c["decay"]
            was[old[s]:] = 0.0
            out[page, h, j % bt] = was + added
    return out


def _grid64(x):
    """Nearest e4m3 values (ties to even) of 64-bit x within +-448."""
    _, e = torch.frexp(x)
    step = _pow2((e - 4).clamp_min(-9)).double()
    return torch.round(x / step) * step


def _evict64(st):
    """The codes' values of both pools."""
    c = st["case"]
    bt = c["bt"]
    out = [st[n].view(torch.float8_e4m3fn).double() for n in ("kp", "vp")]
    before = [x.clone() for x in out]
    lens, keep = st["lens"].tolist(), st["keep"].tolist()
    for s, (length, k) in enumerate(zip(lens, keep)):
        j = torch.arange(length, device=DEV)
        page = st["tables"][s].long()[j // bt]
        last = min(k, c["recent"])
        first = min(k - last, c["sink"])
        for h in range(c["num_kv"]):
            w = st["weights"][page, h, j % bt].double()
            w[:first] = math.inf
            w[length - last:] = math.inf
            rows = torch.argsort(-w, stable=True)[:k].sort().values
            for a in range(0, k, bt):
                r = rows[a:a + bt]
                to = page[a]
                for i, exps in enumerate((st["ke"], st["ve"])):
                    e = exps[page[r], h].double()
                    out[i][to, :len(r), h] = _grid64(before[i][page[r], r % bt, h] * torch.exp2(e - e.max())[:, None])
    return {"k": out[0], "v": out[1], "ke": None, "ve": None, "weights": None, "kept": None}


def _beam64(st):
    """The scores alone: which tokens have them are whole numbers."""
    c = st["case"]
    x = st["logits"].double().log_softmax(-1) + st["scores"].double().view(-1, 1)
    over = st["done"].view(-1) != 0
    x[over] = -math.inf
    x[over, 2] = st["scores"].double().view(-1)[over]
    return {"parents": None, "tokens": None, "scores": x.view(c["n"], -1).topk(c["take"], -1).values}


def exact(case, seed):
    kind = case["kind"]
    if kind == "reorder":
        return None   # whole numbers
    st = prepare(case, seed)
    if kind == "norm":
        return {n: _norm64(st, st[n], st["w" + n]) for n in ("q", "k")}
    if kind == "grad":
        (q, wq), (k, wk) = (_norm64(st, st[n], st["w" + n], st["d" + n]) for n in ("q", "k"))
        return {"q": q, "k": k, "wq": wq, "wk": wk}
    return {"weigh": _weigh64, "evict": _evict64, "beam": _beam64}[kind](st)
