"""Operators of a serving loop with an 8-bit cache, and of layers with local attention, as measurable cases.

    write    keys and values of new tokens quantised into a paged cache, with a scale for each page and head
             (trtamd_kv_cache_write)
    read     tokens of the cache back in FP16 (trtamd_kv_cache_read)
    store    the two behind each other: new tokens written, whole sequences read back
    cached   attention of the newest tokens over their sequences in the cache, causal, with or without a sliding window
             and first tokens that stay visible (trtamd_kv_cache_attention)
    window   attention over packed FP16 sequences with a window on either side and first tokens that stay visible
             (trtamd_window_attention)

`run` computes them in elementary torch operations, or with `own` set through the library.

The cache. Token t of sequence b is token t % page of page table[b][t // page]; keys are [pages][heads][page][d], values
[pages][heads][d][page], in INT8 or E4M3 (top 127 or 448), and a page's keys, or values, of a head share a scale. A page whose first
token is written has the scale max|x| / top; where a page goes on and a new value passes scale * top, the scale doubles until none does
and what the page held is rounded to it. `lengths` counts the tokens of each sequence, those of the call, its last ones, included.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TOP = {"int8": 127.0, "fp8": 448.0}
TRT = {"int8": 2, "fp8": 6}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def _cache(kind, B, new, ctx, **more):
    """`new` tokens of each of B sequences that hold up to `ctx` before them; ragged: both spread over the sequences."""
    case = dict(kind=kind, B=B, new=new, ctx=ctx, kv_heads=8, d=128, page=64, dtype="int8", ragged=False)
    if kind == "cached":
        case.update(heads=32, window=0, sinks=0)
    case.update(more)
    return case


def _window(B, longest, **more):
    """B packed sequences of up to `longest` tokens; left and right: tokens on either side, -1 for all."""
    case = dict(kind="window", B=B, longest=longest, heads=16, kv_heads=16, d=64, left=64, right=64, sinks=0)
    case.update(more)
    return case


def listed():
    return [
        # the next token of one conversation: latency
        dict(name="cache write one token", **_cache("write", 1, 1, 1000, dtype="fp8")),
        # the next token of everyone that a server works for, small pages
        dict(name="cache write batch of 64", **_cache("write", 64, 1, 8000, dtype="fp8", page=16, ragged=True)),
        # prompts of an ordinary batch go into the cache and come back for a layer that works in FP16
        dict(name="cache write and read prompts", **_cache("store", 128, 384, 0, kv_heads=16, d=64, page=32, ragged=True)),
        # one conversation's keys and values in FP16 again, the last page not full
        dict(name="cache read one request", **_cache("read", 1, 777, 0)),
        # the next token of one conversation, heads of their own
        dict(name="cache attention one token", **_cache("cached", 1, 1, 1000, heads=16, kv_heads=16, d=64)),
        # the next token of everyone that a server works for
        dict(name="cache attention batch of 64", **_cache("cached", 64, 1, 8000, dtype="fp8", page=16, ragged=True)),
        # one conversation far into its context
        dict(name="cache attention long context", **_cache("cached", 1, 1, 131070)),
        # two drafted tokens and the next one each, local layers with the first tokens visible
        dict(name="cache attention drafts in window",
             **_cache("cached", 32, 3, 20000, page=32, window=4096, sinks=4, ragged=True)),
        # a piece of each of four long prompts behind what the cache has of them
        dict(name="cache attention prompt pieces", **_cache("cached", 4, 1024, 8192, dtype="fp8")),
        # one short request through a local encoder layer
        dict(name="window attention one request", **_window(1, 77, heads=12, kv_heads=12)),
        # the benchmark batch through a local encoder layer
        dict(name="window attention batch of 128", **_window(128, 384)),
        # a document through a local causal layer with shared keys and visible first tokens
        dict(name="window attention document", **_window(1, 8001, kv_heads=4, d=128, left=1023, right=0, sinks=4)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "store", "read", "cached", "cached", "cached", "window", "window"))
    if kind == "window":
        while True:
            B, longest, heads = _log(rng, 1, 128), _log(rng, 1, 8001), rng.choice((4, 8, 12, 16))
            if B * longest * longest * heads <= 8001 * 8001 * 16 and B * longest <= 50000:
                break
        causal, reach = rng.random() < 0.4, _log(rng, 1, 4096)
        return _window(B, longest, heads=heads, kv_heads=rng.choice((heads, heads // 4)), d=rng.choice((32, 64, 64, 80, 96, 128, 128)),
                       left=rng.choice((reach, reach, -1)), right=0 if causal else rng.choice((reach, 2 * reach, -1)),
                       sinks=rng.choice((0, 0, 1, 4, 70)))
    more = dict(d=rng.choice((64, 64, 80, 96, 128, 128)), page=rng.choice((16, 32, 64, 128)), dtype=rng.choice(("int8", "fp8")),
                kv_heads=rng.choice((1, 4, 8, 12)), ragged=rng.random() < 0.7)
    if kind == "write":
        more["dtype"] = "fp8"  # its codes are values by themselves
    while True:
        B, ctx = _log(rng, 1, 64), _log(rng, 1, 131070) if kind != "read" else 0
        new = _log(rng, 1, 1024) if kind == "read" or rng.random() < 0.4 else rng.choice((1, 1, 2, 5))
        if kind == "cached":
            more.update(heads=more["kv_heads"] * rng.choice((1, 2, 4, 7, 8)), window=rng.choice((0, 0, _log(rng, 16, 8192))),
                        sinks=rng.choice((0, 4, 17)))
            if B * new * more["heads"] * (ctx + new) > 4 * 1024 * 32 * 9216 / 4:
                continue
        if B * (ctx + new) * more["kv_heads"] * more["d"] <= 64 * 8000 * 8 * 128 / 2:
            break
    return _cache(kind, B, new, ctx, **more)


# ---- inputs ------------------------------------------------------------------------------------------------------

def _spread(n, top, ragged):
    """n whole numbers up to `top`, the first of them `top` itself; ragged: spread from a twentieth on."""
    r = np.random.default_rng(n)
    a = np.round(np.exp(r.uniform(math.log(max(1, top // 20)), math.log(max(1, top)), n))).astype(np.int64)
    a[0] = top
    return np.minimum(a, top) if ragged else np.full(n, top)


def _new_and_lengths(case):
    """The call's tokens of each sequence, and its tokens with what the cache had before them."""
    new = _spread(case["B"], case["new"], case["ragged"] and case["new"] > 5)
    return new, new + (_spread(case["B"], case["ctx"], case["ragged"])[::-1] if case["ctx"] else 0)


def _prepare_cache(case, seed):
    B, H, d, P, top = case["B"], case["kv_heads"], case["d"], case["page"], TOP[case["dtype"]]
    g, r = torch.Generator(device=DEVICE).manual_seed(seed), np.random.default_rng(seed)
    mixed = r.permutation(B)
    new, lengths = (n[mixed] for n in _new_and_lengths(case))
    pages_of = -(-lengths // P)
    pages = int(pages_of.sum()) + 3
    # pages were handed out as they came free: in no order
    order, table, at = r.permutation(pages), np.full((B, int(pages_of.max()) + 1), -1), 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    rand = lambda *s: torch.randn(s, generator=g, device=DEVICE)
    state = dict(kind=case["kind"], dtype=case["dtype"], P=P, H=H, d=d, B=B, most=int(new.max()), longest=int(lengths.max()),
                 table=torch.from_numpy(table.astype(np.int32)).to(DEVICE), lengths=torch.from_numpy(lengths.astype(np.int32)).to(DEVICE),
                 cu=torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEVICE))
    T = int(new.sum())
    # what earlier calls left: a page's largest of P * d normal values is 3 to 4 deviations
    for name, shape in (("k", (pages, H, P, d)), ("v", (pages, H, d, P))):
        codes = (rand(*shape) * (top / 3.5)).clamp_(-top, top)
        state[name] = (codes.round_() if case["dtype"] == "int8" else codes).to(CODES[case["dtype"]])
        state[name + "_scale"] = 3.5 / top * torch.exp(0.3 * rand(pages, H))
        del codes
    if case["kind"] in ("write", "store"):
        # the projection's result: [token][head][k|v][d], some tokens louder than the rest
        kv = (rand(T, H, 2, d) * torch.exp(0.5 * rand(T, 1, 1, 1))).half()
        state.update(new_k=kv[:, :, 0], new_v=kv[:, :, 1])
    if case["kind"] in ("read", "store"):  # whole sequences come back
        state.update(cu_read=torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).to(DEVICE), T_read=int(lengths.sum()))
    if case["kind"] == "cached":
        state.update(q=rand(T, case["heads"], d).half(), scale=1 / math.sqrt(d), window=case["window"], sinks=case["sinks"])
    return state


def _prepare_window(case, seed):
    H, Hk, d = case["heads"], case["kv_heads"], case["d"]
    g, r = torch.Generator(device=DEVICE).manual_seed(seed), np.random.default_rng(seed)
    lens = r.permutation(_spread(case["B"], case["longest"], case["B"] > 1))
    T = int(lens.sum())
    qkv = torch.randn((T, H + 2 * Hk, d), generator=g, device=DEVICE).half()
    if H == Hk:  # the packing of the attention plugins
        by_head = qkv.view(T, H, 3, d)
        q, k, v = by_head[:, :, 0], by_head[:, :, 1], by_head[:, :, 2]
    else:
        q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    return dict(kind="window", q=q, k=k, v=v, cu=torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).to(DEVICE),
                B=case["B"], longest=case["longest"], scale=1 / math.sqrt(d), left=case["left"], right=case["right"], sinks=case["sinks"])


def prepare(case, seed):
    return (_prepare_window if case["kind"] == "window" else _prepare_cache)(case, seed)


# ---- the operators through the library ---------------------------------------------------------------------------

def _described(capi, state, cu, T, most):
    c = capi.KvCache()
    c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lengths = (
        state[n].data_ptr() for n in ("k", "v", "k_scale", "v_scale", "table", "lengths"))
    c.cu_seqlens, c.T, c.max_tokens, c.data_type = cu.data_ptr(), T, most, TRT[state["dtype"]]
    c.B, c.max_pages, c.pages, c.page_tokens = state["B"], state["table"].shape[1], state["k"].shape[0], state["P"]
    c.kv_heads, c.d = state["H"], state["d"]
    return c


def _strided(p, name, t):
    setattr(p, name, t.data_ptr())
    setattr(p, name + "_token_stride", t.stride(0))
    setattr(p, name + "_head_stride", t.stride(1))


def _bind(state):
    """The calls as a program keeps them from pass to pass: their parameters, outputs and workspaces."""
    from tensorrt_amd import capi
    api, calls = capi.api(), []
    kept = state["kept"] = []
    half = lambda *s: torch.empty(s, dtype=torch.float16, device=DEVICE)

    def call(function, p):
        kept.append(p)
        calls.append((function, ctypes.byref(p)))

    if state["kind"] == "window":
        q, k, v = state["q"], state["k"], state["v"]
        out = half(*q.shape)
        p = capi.WindowAttentionParams()
        for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
            _strided(p, name, t)
        p.cu_seqlens, p.B, p.T, p.max_tokens = state["cu"].data_ptr(), state["B"], q.shape[0], state["longest"]
        p.q_heads, p.kv_heads, p.d = q.shape[1], k.shape[1], q.shape[2]
        p.scale, p.left, p.right, p.sinks = state["scale"], state["left"], state["right"], state["sinks"]
        call(api.window_attention, p)
        state["result"] = out
    if state["kind"] in ("write", "store"):
        p = capi.KvCacheWriteParams()
        p.cache = _described(capi, state, state["cu"], state["new_k"].shape[0], state["most"])
        _strided(p, "k", state["new_k"])
        _strided(p, "v", state["new_v"])
        call(api.kv_cache_write, p)
        state["result"] = tuple(state[n] for n in ("k", "v", "k_scale", "v_scale"))
    if state["kind"] in ("read", "store"):
        outs = tuple(half(state["T_read"], state["H"], state["d"]) for _ in range(2))
        p = capi.KvCacheReadParams()
        p.cache = _described(capi, state, state["cu_read"], state["T_read"], state["longest"])
        _strided(p, "k", outs[0])
        _strided(p, "v", outs[1])
        call(api.kv_cache_read, p)
        state["result"] = outs if state["kind"] == "read" else outs + (state["k_scale"], state["v_scale"])
    if state["kind"] == "cached":
        q, out = state["q"], half(*state["q"].shape)
        p = capi.KvCacheAttentionParams()
        p.cache = _described(capi, state, state["cu"], q.shape[0], state["most"])
        _strided(p, "q", q)
        _strided(p, "out", out)
        p.q_heads, p.scale, p.window, p.sinks, p.max_length = q.shape[1], state["scale"], state["window"], state["sinks"], state["longest"]
        size = api.kv_cache_attention_workspace_size(ctypes.byref(p))
        kept.append(torch.empty((max(size, 16),), dtype=torch.uint8, device=DEVICE))
        p.workspace, p.workspace_bytes = kept[-1].data_ptr(), size
        call(api.kv_cache_attention, p)
        state["result"] = out
    state["calls"], state["check"] = calls, api.check


def _run_own(state):
    if "calls" not in state:
        _bind(state)
    stream = torch.cuda.current_stream().cuda_stream
    for function, p in state["calls"]:
        state["check"](function(stream, p))
    return state["result"]


# ---- the same in elementary operations, binary32 -----------------------------------------------------------------

def _bytes(codes):
    return codes.view(torch.int8)


def _rounded(y, dtype):
    """y, within the type's range, as the nearest codes."""
    top = TOP[dtype]
    y = y.clamp(-top, top)
    return (y.round() if dtype == "int8" else y).to(CODES[dtype])


def _run_write(state):
    P, H, d, dtype = state["P"], state["H"], state["d"], state["dtype"]
    top = TOP[dtype]
    cu, end, table = state["cu"].long(), state["lengths"].long(), state["table"].long()
    begin = end - (cu[1:] - cu[:-1])
    first = begin // P
    blocks = (state["most"] + P - 2) // P + 1  # pages that a sequence's new tokens can touch
    block = first[:, None] + torch.arange(blocks, device=DEVICE)
    touched = block * P < end[:, None]
    page = table.gather(1, block.clamp(max=table.shape[1] - 1))[touched]
    at = block[..., None] * P + torch.arange(P, device=DEVICE)
    fresh = ((at >= begin[:, None, None]) & (at < end[:, None, None]))[touched]
    before = (at < begin[:, None, None])[touched]
    row = (cu[:-1, None, None] + at - begin[:, None, None])[touched].clamp(0, int(state["new_k"].shape[0]) - 1)
    for name in ("k", "v"):
        x = torch.where(fresh[..., None, None], state["new_" + name].float()[row], 0.0).permute(0, 2, 1, 3)  # [block][head][token][d]
        amax = x.abs().amax((2, 3))
        old = torch.where(before.any(1)[:, None], state[name + "_scale"][page], 0.0)
        limit = old * top
        m0, e0 = torch.frexp(amax)
        m1, e1 = torch.frexp(limit)
        doublings = torch.where((limit > 0) & (amax > limit), e0 - e1 + (m0 > m1), 0)
        scale = torch.where(limit > 0, torch.ldexp(old, doublings), amax / top)
        inverse = torch.where(scale > 0, 1 / scale, 0.0)
        codes = _rounded(x * inverse[..., None, None], dtype)
        held = state[name][page] if name == "k" else state[name][page].view(torch.int8).transpose(2, 3).contiguous().view(CODES[dtype])
        again = _rounded(torch.ldexp(held.float(), -doublings[..., None, None]), dtype)
        was = before[:, None, :, None] & (doublings > 0)[..., None, None]
        both = torch.where(fresh[:, None, :, None], _bytes(codes), torch.where(was, _bytes(again), _bytes(held)))
        _bytes(state[name])[page] = both if name == "k" else both.transpose(2, 3)
        state[name + "_scale"][page] = scale
    return tuple(state[n] for n in ("k", "v", "k_scale", "v_scale"))


def _gathered(state, name, page, slot):
    """Keys or values of the tokens `slot` of the pages `page`, and their scales."""
    codes = _bytes(state[name])
    codes = codes[page, :, slot] if name == "k" else codes[page, :, :, slot]
    return codes.view(CODES[state["dtype"]]).float() * state[name + "_scale"][page][..., None]


def _run_read(state):
    cu, P = state["cu_read"].long(), state["P"]
    token = torch.arange(state["T_read"], device=DEVICE)
    b = torch.searchsorted(cu, token, right=True) - 1
    at = token - cu[b]
    page = state["table"].long()[b, at // P]
    return tuple(_gathered(state, n, page, at % P).half() for n in ("k", "v"))


def _attend(q, k, v, visible, scale):
    """q [B][n][heads][d], k and v [B][keys][kv heads][d], visible [B][n][keys]: the context, 0 where nothing is visible."""
    B, n, heads, d = q.shape
    H = k.shape[2]
    group = heads // H
    q = q.view(B, n, H, group, d).permute(0, 2, 3, 1, 4).reshape(B, H, group * n, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(B, H, group, n, -1).mul_(scale)
    s.masked_fill_(~visible[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, group * n, -1), v.transpose(1, 2).contiguous()).view(B, H, group, n, d)
    return torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, heads, d)


def _padded_rows(cu, n):
    """Which row of a packed tensor token i of each sequence is, and whether there is one."""
    i = torch.arange(n, device=DEVICE)
    lens = cu[1:] - cu[:-1]
    return (cu[:-1, None] + i).clamp(max=int(n * len(lens))), i < lens[:, None]


def _run_cached(state):
    P, n, L = state["P"], state["most"], state["longest"]
    cu, end, table = state["cu"].long(), state["lengths"].long(), state["table"].long()
    j = torch.arange(L, device=DEVICE)
    there = j < end[:, None]
    page = table[:, j // P].clamp(min=0)
    slot = (j % P).expand(state["B"], L)
    k, v = (torch.where(there[..., None, None], _gathered(state, name, page, slot), 0.0) for name in ("k", "v"))
    row, real = _padded_rows(cu, n)
    q = state["q"].float()
    at = (end - (cu[1:] - cu[:-1]))[:, None] + torch.arange(n, device=DEVICE)
    near = j > at[..., None] - (state["window"] or L)
    visible = (j <= at[..., None]) & (near | (j < state["sinks"])) & there[:, None]
    out = _attend(q[row.clamp(max=q.shape[0] - 1)], k, v, visible, state["scale"])
    return out[real].half()


def _run_window(state):
    cu, n = state["cu"].long(), state["longest"]
    row, real = _padded_rows(cu, n)
    row = row.clamp(max=state["q"].shape[0] - 1)
    q, k, v = (state[name].float()[row] for name in ("q", "k", "v"))
    j = torch.arange(n, device=DEVICE)
    off = j - j[:, None]
    left, right = (n if state[side] < 0 else state[side] for side in ("left", "right"))
    near = ((off >= -left) | (j < state["sinks"])) & (off <= right)
    return _attend(q, k, v, near & real[:, None], state["scale"])[real].half()


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "window":
        return _run_window(state)
    if state["kind"] == "cached":
        return _run_cached(state)
    written = _run_write(state) if state["kind"] != "read" else ()
    return written if state["kind"] == "write" else _run_read(state) + written[2:]


# ---- the definitions in binary64 ---------------------------------------------------------------------------------

def _exact_codes(x, dtype):
    """Real numbers to the values of the nearest codes."""
    top = TOP[dtype]
    x = x.clamp(-top, top)
    if dtype == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)  # three bits behind the leading one
    return (x / step).round() * step


def _exact_write(state):
    """Page by page. The codes as real numbers, [pages][heads][page][d] both, and the scales."""
    P, dtype = state["P"], state["dtype"]
    cu, lengths, table = (state[n].cpu().numpy() for n in ("cu", "lengths", "table"))
    found = {}
    for name in "kv":
        codes = state[name].double() if name == "k" else state[name].double().transpose(2, 3).contiguous()
        scales, new = state[name + "_scale"].double().clone(), state["new_" + name].double()
        for b in range(state["B"]):
            end, n = int(lengths[b]), int(cu[b + 1] - cu[b])
            for block in range((end - n) // P, -(-end // P)):
                lo, hi = max(end - n, block * P), min(end, block * P + P)
                x, page = new[int(cu[b]) + lo - (end - n):int(cu[b]) + hi - (end - n)].transpose(0, 1), int(table[b, block])
                peak, here = x.abs().amax((1, 2)), slice(lo - block * P, hi - block * P)
                if here.start and bool((scales[page] > 0).all()):
                    times = torch.ceil(torch.log2(peak / (scales[page] * TOP[dtype]))).clamp_min(0)
                    codes[page, :, :here.start] = _exact_codes(codes[page, :, :here.start] / torch.exp2(times)[:, None, None], dtype)
                    scales[page] *= torch.exp2(times)
                else:
                    scales[page] = peak / TOP[dtype]
                codes[page, :, here] = _exact_codes(x / scales[page][:, None, None], dtype)
        found[name], found[name + "_scale"] = codes, scales
    return found


def _exact_sequences(state, found, name):
    """Each sequence's keys or values, [tokens][heads][d]."""
    P, lengths = state["P"], state["lengths"].cpu().numpy()
    for b in range(state["B"]):
        page = state["table"][b, :-(-int(lengths[b]) // P)].long()
        if found is None:
            codes = state[name][page].double()
            x = (codes if name == "k" else codes.transpose(2, 3)) * state[name + "_scale"].double()[page, :, None, None]
        else:
            x = found[name][page] * found[name + "_scale"][page, :, None, None]
        yield x.transpose(1, 2).flatten(0, 1)[:int(lengths[b])]


def _exact_attention(q, k, v, scale, visible):
    """One sequence, head by head."""
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    for h in range(q.shape[1]):
        s = torch.addmm(torch.zeros((), dtype=torch.float64, device=DEVICE), q[:, h].double(), k[:, h // group].double().t().contiguous(), beta=0, alpha=scale)
        w = torch.softmax(s.masked_fill(~visible, -math.inf), 1).nan_to_num(0.0)
        out[:, h] = torch.mm(w, v[:, h // group].double().contiguous())
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind in ("write", "store"):
        found = _exact_write(state)
        if kind == "write":
            return found["k"], found["v"].transpose(2, 3).contiguous(), found["k_scale"], found["v_scale"]
        return tuple(torch.cat(list(_exact_sequences(state, found, n))) for n in "kv") + (found["k_scale"], found["v_scale"])
    if kind == "read":
        return tuple(torch.cat(list(_exact_sequences(state, None, n))) for n in "kv")
    cu, outs = state["cu"].cpu().numpy(), []
    if kind == "cached":
        for b, (k, v) in enumerate(zip(_exact_sequences(state, None, "k"), _exact_sequences(state, None, "v"))):
            q, j = state["q"][int(cu[b]):int(cu[b + 1])], torch.arange(k.shape[0], device=DEVICE)
            back = torch.arange(k.shape[0] - q.shape[0], k.shape[0], device=DEVICE)[:, None] - j
            visible = back >= 0
            if case["window"]:
                visible &= (back < case["window"]) | (j < case["sinks"])
            outs.append(_exact_attention(q, k, v, state["scale"], visible))
    else:
        for lo, hi in zip(cu[:-1], cu[1:]):
            j = torch.arange(int(hi - lo), device=DEVICE)
            back = j[:, None] - j
            visible = torch.ones_like(back, dtype=torch.bool)
            if case["left"] >= 0:
                visible &= (back <= case["left"]) | (j < case["sinks"])
            if case["right"] >= 0:
                visible &= back >= -case["right"]
            outs.append(_exact_attention(*(state[n][int(lo):int(hi)] for n in "qkv"), state["scale"], visible))
    return torch.cat(outs)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _visible(n, L, left, right, sinks):
    """Keys that the last n of L tokens see, all together, and keys that any of them sees."""
    at = np.arange(L - n, L)
    hi = np.minimum(at + right + 1, L) if right >= 0 else np.full(n, L)
    lo = np.maximum(at - left, 0) if left >= 0 else np.zeros(n, np.int64)
    first = np.minimum(np.minimum(sinks, lo), hi)
    return int((hi - lo + first).sum()), int(hi.max() - lo.min() + first.min())


def work(case):
    if case["kind"] == "window":
        lens = _spread(case["B"], case["longest"], case["B"] > 1)
        pairs = sum(_visible(int(n), int(n), case["left"], case["right"], case["sinks"])[0] for n in lens)
        return dict(bytes=4 * int(lens.sum()) * (case["heads"] + case["kv_heads"]) * case["d"], flops=4 * pairs * case["heads"] * case["d"])
    values = case["kv_heads"] * case["d"]
    new, lengths = _new_and_lengths(case)
    T, tokens = int(new.sum()), int(lengths.sum())
    writes, reads = T * values * 2 * 3, tokens * values * 2 * 3
    if case["kind"] != "cached":
        bytes_ = {"write": writes, "read": reads, "store": writes + reads}[case["kind"]]
        return dict(bytes=bytes_, flops=bytes_)
    counts = [_visible(int(n), int(L), case["window"] - 1, 0, case["sinks"]) for n, L in zip(new, lengths)]
    return dict(bytes=2 * values * sum(c[1] for c in counts) + 4 * T * case["heads"] * case["d"],
                flops=4 * case["heads"] * case["d"] * sum(c[0] for c in counts))
