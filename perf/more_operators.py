"""Performance cases of serving from an 8-bit paged KV cache: what a step of a
server calls beside the QMatMuls where the cache holds one byte a value.

  plan     pages of the pool for the tokens that each sequence of the batch asks
           for or drops: page table, lengths, ranges of packed rows, slot map
  append   RoPE of the packed q and k rows; k and v into the cache's pages as
           e4m3 codes with a power of two for each 16 positions of a head
  decode   attention of one new token per sequence over the pages
  prefill  causal attention of packed prompt rows (or of a chunk of a prompt
           whose earlier part is cached already) over the pages

Layer shapes are a 7B decoder's (32 heads of 128) and generic grouped-head ones;
``draw`` covers the same kinds over smaller, odd and ragged sizes.  q, k and v are
N(0, 1) rows as a norm and a projection leave them, keys and values with a
magnitude of each head's own, and the pages of a sequence are scattered over the
pool as an allocator leaves them after some hours.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # False: the plain forms; True: the package's kernels

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 16  # positions of a head that share a scale
CODE, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---- cases ----
# n_seqs sequences; their lengths before the call are spread between past_lo and
# past_hi and their new rows between new_lo and new_hi (over the logarithm, by
# `mix`); every `idle`-th slot of the batch holds no sequence (0: none).  plan: every
# `ended`-th sequence has ended and gives its pages back, the one after it drops its
# last 5 tokens; the pool has `pool` per cent of the pages that the batch asks for.

def listed():
    seven = {"heads": 32, "kv_heads": 32, "dim": 128, "act": "f32", "page": 16, "mix": 1, "idle": 0}
    grouped = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "mix": 2, "idle": 0}
    one = {"new_lo": 1, "new_hi": 1}
    return [
        # a decode step of a serving batch: one token each, some sequences end
        {"name": "plan_step", "kind": "plan", "seqs": 256, "page": 16, "mix": 1, "idle": 29, "past_lo": 8,
         "past_hi": 8000, "ended": 17, "pool": 130, **one},
        # a large step of prompts and single tokens together, more asked for than the pool has
        {"name": "plan_mixed", "kind": "plan", "seqs": 1500, "page": 16, "mix": 2, "idle": 7, "past_lo": 0,
         "past_hi": 2000, "new_lo": 1, "new_hi": 700, "ended": 13, "pool": 60},
        # one token of one sequence of a 7B decoder: the smallest append
        dict(seven, name="append_token", kind="append", seqs=1, past_lo=700, past_hi=700, **one),
        # one token each of a large batch, bf16 activations
        dict(grouped, name="append_batch", kind="append", act="bf16", seqs=256, past_lo=8, past_hi=1000, **one),
        # a packed batch of ragged prompts, f32 projections as frq_qmatmul writes them
        dict(grouped, name="append_prompts", kind="append", act="f32", seqs=21, past_lo=0, past_hi=90, new_lo=40,
             new_hi=1900),
        # one token of a 7B decoder after a conversation of 900: the smallest attention
        dict(seven, name="decode_token", kind="decode", seqs=1, past_lo=900, past_hi=900, **one),
        # one sequence with a very long context: the split over the length
        dict(grouped, name="decode_long", kind="decode", act="f16", seqs=1, past_lo=200001, past_hi=200001, **one),
        # a serving batch of mixed lengths with idle slots, f32 activations (frq_qmatmul's output)
        dict(grouped, name="decode_ragged", kind="decode", act="f32", seqs=96, past_lo=30, past_hi=8000, idle=11, **one),
        # many sequences of a model with heads of 64, larger pages
        dict(grouped, name="decode_dim64", kind="decode", heads=64, dim=64, act="bf16", seqs=128, past_lo=300,
             past_hi=2500, page=64, mix=4, **one),
        # a packed batch of ragged prompts
        dict(grouped, name="prefill_ragged", kind="prefill", act="f16", seqs=15, past_lo=0, past_hi=0, new_lo=60,
             new_hi=1900, mix=5),
        # one long prompt
        dict(grouped, name="prefill_long", kind="prefill", act="bf16", seqs=1, past_lo=0, past_hi=0, new_lo=12345,
             new_hi=12345),
        # a chunk of a 7B decoder's prompt after its cached part, f32 activations
        dict(seven, name="prefill_chunk", kind="prefill", seqs=2, past_lo=3500, past_hi=7000, new_lo=300, new_hi=512),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["plan", "append", "decode", "decode", "prefill", "prefill"])
    case = {"kind": kind, "page": rng.choice([16, 16, 32, 64, 256]), "mix": rng.randint(1, 10 ** 6),
            "idle": rng.choice([0, 0, 3, 7])}
    if kind == "plan":
        seqs, past = _log(rng, 1, 3000), _log(rng, 1, 4000)
        new = rng.choice([1, _log(rng, 1, max(1, 200000 // seqs))])
        return dict(case, seqs=seqs, past_lo=rng.randint(0, past), past_hi=past, new_lo=1, new_hi=new,
                    ended=rng.choice([0, 3, 20]), pool=rng.choice([60, 100, 150]))
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (16, 2), (8, 1), (28, 4), (40, 8), (64, 8), (20, 1)])
    case.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([128, 128, 64]), act=rng.choice(["f32", "f16", "bf16"]))
    if kind == "decode":
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, min(200000, (200 << 20) // (kv_heads * case["dim"] * seqs))))
        return dict(case, seqs=seqs, past_lo=rng.randint(0, hi), past_hi=hi, new_lo=1, new_hi=1)
    if kind == "append":
        seqs = _log(rng, 1, 256)
        new = rng.choice([1, _log(rng, 1, max(1, 16384 // seqs))])
        past = _log(rng, 1, 512)
        return dict(case, seqs=seqs, past_lo=rng.randint(0, past), past_hi=past, new_lo=_log(rng, 1, new), new_hi=new)
    seqs = _log(rng, 1, 32)
    # the plain form's scores: seqs * rows * length * heads values at most
    most = 12345 * 6000 // seqs * 32 // heads
    new = _log(rng, 1, min(6000, math.isqrt(most)))
    past = rng.choice([0, _log(rng, 1, max(1, min(16384, most // new - new)))])
    return dict(case, seqs=seqs, past_lo=rng.randint(0, past), past_hi=past, new_lo=_log(rng, 1, new), new_hi=new)


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return lo if lo == hi else min(hi, max(lo, _log(rng, max(1, lo), hi)))


def _lengths(case):
    """(rows, kv_len) of every slot: host lists, by the case alone.  plan: the
    tokens asked for (below 0: dropped), and the lengths before the call."""
    rng = random.Random(case["mix"])
    rows, kv = [], []
    for s in range(case["seqs"]):
        new, past = _spread(rng, case["new_lo"], case["new_hi"]), _spread(rng, case["past_lo"], case["past_hi"])
        idle = case["idle"] and s % case["idle"] == case["idle"] - 1
        if case["kind"] == "plan":
            ended = case["ended"] and s % case["ended"]
            rows.append(0 if idle else -past if ended == 1 else -5 if ended == 2 else new)
            kv.append(0 if idle else past)
        elif case["kind"] == "decode":  # one row a slot, also where it is idle
            rows.append(1)
            kv.append(0 if idle else past + new)
        else:
            rows.append(0 if idle else new)
            kv.append(0 if idle else past + new)
    if case["kind"] != "plan" and not sum(rows):
        rows[0], kv[0] = 1, 1
    return rows, kv


def _pages(n: int, case) -> int:
    return -(-n // case["page"])


def _plan_sizes(case):
    """(max_pages, pages of the pool, rows of the packed arrays): a padded batch."""
    tokens, kv = _lengths(case)
    asked = sum(_pages(k + t, case) - _pages(k, case) for t, k in zip(tokens, kv) if t > 0)
    rows = sum(t for t in tokens if t > 0)
    return (max(_pages(k + max(t, 0), case) for t, k in zip(tokens, kv)) + 1,
            sum(_pages(k, case) for k in kv) + max(1, asked * case["pool"] // 100), rows + rows // 16 + 8)


def work(case):
    rows, kv = _lengths(case)
    if case["kind"] == "plan":
        moved = sum(abs(_pages(max(0, k + t), case) - _pages(k, case)) for t, k in zip(rows, kv))
        # tokens and lengths in, lengths and row ranges out; a page id read and written; slot and position
        return {"bytes": 16 * len(kv) + 8 * moved + 12 * _plan_sizes(case)[2], "flops": 0}
    a, d = SIZE[case["act"]], case["dim"]
    h, hk = case["heads"], case["kv_heads"]
    n = sum(rows)
    if case["kind"] == "append":
        positions, blocks = set(), 0
        for r, k in zip(rows, kv):
            positions.update(range(k - r, k))
            blocks += (k - 1) // BLOCK - (k - r) // BLOCK + 1 if r else 0
        # q read and written, k and v read and their codes and scales written, the tables' rows
        return {"bytes": n * (2 * h * d * a + 2 * hk * d * (a + 1)) + 2 * blocks * hk + len(positions) * 2 * d * 4,
                "flops": 5 * n * (h + hk) * d}
    # codes and scales of every sequence once, q and out once; two products per visible pair
    pairs = sum(r * k - r * (r - 1) // 2 for r, k in zip(rows, kv) if k)
    scales = sum(-(-k // BLOCK) for k in kv)
    return {"bytes": 2 * hk * (sum(kv) * d + scales) + 2 * n * h * d * a, "flops": 4 * h * d * pairs}


# ---- inputs ----

def _power(e):
    """2^e of whole numbers -127 .. 127, exactly, in f32."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _exponent(amax):
    """The least e of -127 .. 120 for which amax <= 448 * 2^e (448: e4m3's largest)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 8 - (m <= 0.875).to(torch.int32), -127).clamp(-127, 120)


def _encode(x):
    """Codes and scales of blocks [..., BLOCK, d] of f32 values."""
    e = _exponent(x.abs().amax((-2, -1)))
    return (x * _power(-e)[..., None, None]).to(CODE), (e + 127).to(torch.uint8)


def prepare(case, seed):
    if own:
        _one_stream()
    g = torch.Generator("cuda").manual_seed(seed)
    rng = random.Random(seed)
    rows, kv = _lengths(case)
    ps = case["page"]
    need = [_pages(k, case) for k in kv]
    width, n_pages, n = max(max(need), 1), sum(need) + 7, sum(rows)
    if case["kind"] == "plan":
        width, n_pages, n = _plan_sizes(case)
    order = list(range(n_pages))
    rng.shuffle(order)
    table = torch.zeros(len(kv), width, dtype=torch.int32)
    at = 0
    for s, used in enumerate(need):
        table[s, :used] = torch.tensor(order[at:at + used], dtype=torch.int32)
        at += used

    def ints(*a, dtype=torch.int32):
        return torch.tensor(a, dtype=dtype, device="cuda")

    state = {"case": case, "table": table.cuda(), "kv_len": ints(*kv), "rows": n, "n_pages": n_pages}
    if case["kind"] == "plan":
        free = torch.zeros(n_pages, dtype=torch.int32)
        free[:n_pages - at] = torch.tensor(order[at:], dtype=torch.int32)
        state.update(tokens=ints(*rows), free=free.cuda(), n_free=ints(n_pages - at),
                     kv_out=ints(*[0] * len(kv)), n_free_out=ints(0), start=ints(*[0] * (len(kv) + 1)),
                     slots=torch.zeros(n, dtype=torch.int64, device="cuda"),
                     positions=torch.zeros(n, dtype=torch.int32, device="cuda"))
        if own:
            state["handle"] = _handle(state)
        return state
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    act = TORCH[case["act"]]
    start = [0]
    for r in rows:
        start.append(start[-1] + r)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    size = (0.7 * normal(2, hk)).exp()  # a magnitude of keys and values for each head
    for i, name in enumerate("kv"):
        blocks = normal(n_pages, hk, ps // BLOCK, BLOCK, d) * size[i, :, None, None, None]
        codes, scales = _encode(blocks)
        state[name + "_pages"], state[name + "_scales"] = codes.view(n_pages, hk, ps, d), scales.view(SCALE)
        del blocks
    state.update(scale=1.0 / math.sqrt(d), max_kv_len=max(kv), start=ints(*start),
                 out=torch.empty(n, h * d, dtype=act, device="cuda"))
    if case["kind"] == "append":
        # q, k and v as one projection leaves them: a row of each token, one after the other
        qkv = normal(n, (h + 2 * hk) * d)
        for i in range(2):
            part = qkv[:, (h + i * hk) * d:(h + (i + 1) * hk) * d]
            part.copy_((part.view(n, hk, d) * size[i, :, None]).view(n, hk * d))
        qkv = qkv.to(act)
        state.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + hk) * d], v=qkv[:, (h + hk) * d:])
        angle = torch.arange(max(kv), dtype=torch.float64)[:, None] * \
            10000.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64) / d)
        state.update(cos=torch.cat([angle.cos()] * 2, 1).float().cuda(), sin=torch.cat([angle.sin()] * 2, 1).float().cuda())
    else:
        state["q"] = normal(n, h * d).to(act)
    if own:
        state["handle"] = _handle(state)
    return state


# ---- the package's operators ----

_device = _stream = None


def _one_stream():
    """torch's work and the package's on one stream, so that each waits for what
    the other did before: the device adopts a stream of torch's, which becomes the
    current one (torch's default stream has no handle to adopt)."""
    import fuel_amd as F

    global _device, _stream
    if _device is None:
        _device, _stream = F.RocmDevice(0), torch.cuda.Stream()
        _device.set_stream(_stream.cuda_stream)
    if torch.cuda.current_stream() != _stream:
        _stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(_stream)


def _handle(state):
    """The cache, the batch and the workspace a serving program keeps."""
    import fuel_amd as F

    case = state["case"]
    if case["kind"] == "plan":
        return F, None, None, None, None
    cache = F.PagedKvCache8(_device, state["n_pages"], case["page"], case["kv_heads"], case["dim"],
                            k=state["k_pages"].data_ptr(), v=state["v_pages"].data_ptr(),
                            k_scale=state["k_scales"].data_ptr(), v_scale=state["v_scales"].data_ptr())
    batch = F.PagedBatch(state["table"].data_ptr(), state["kv_len"].data_ptr(), case["seqs"],
                         state["table"].shape[1], state["q"].shape[0],
                         row_start=None if case["kind"] == "decode" else state["start"].data_ptr(),
                         max_kv_len=state["max_kv_len"])
    work = None
    if case["kind"] != "append":
        work = _device.alloc((max(1, F.paged_attention_workspace(cache, batch, case["heads"])),), "uint8")
    return F, cache, batch, {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}[case["act"]], work


def _run_own(state):
    F, cache, batch, act, work = state["handle"]
    case = state["case"]
    if case["kind"] == "plan":
        F.paged_plan(_device, case["seqs"], state["table"].shape[1], case["page"], state["n_pages"], state["rows"],
                     state["tokens"].data_ptr(), state["kv_len"].data_ptr(), state["table"].data_ptr(),
                     state["free"].data_ptr(), state["n_free"].data_ptr(), state["start"].data_ptr(),
                     slots=state["slots"].data_ptr(), positions=state["positions"].data_ptr(),
                     kv_len_out=state["kv_out"].data_ptr(), n_free_out=state["n_free_out"].data_ptr())
        return _planned(state)
    q, out = state["q"], state["out"]
    if case["kind"] == "append":
        F.paged_append(cache, batch, act, case["heads"], q.data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(),
                       out.data_ptr(), ldq=q.stride(0), ldk=state["k"].stride(0), ldv=state["v"].stride(0),
                       rope_cos=state["cos"].data_ptr(), rope_sin=state["sin"].data_ptr(), rope_rows=state["cos"].shape[0])
        return _appended(state)
    attend = F.paged_attention_decode if case["kind"] == "decode" else F.paged_attention_prefill
    attend(cache, batch, act, case["heads"], q.data_ptr(), out.data_ptr(), state["scale"], work)
    return out


def _planned(state):
    return {k: state[k] for k in ("table", "kv_out", "free", "n_free_out", "start", "slots", "positions")}


def _appended(state):
    """Rotated q, and the cache as the numbers that its bytes stand for: codes in
    units of their block's scale, and the scales."""
    return {k: state[k] for k in ("out", "k_pages", "v_pages", "k_scales", "v_scales")}


# ---- the plain forms ----

def _plain_plan(state):
    ps = state["case"]["page"]
    tokens, kv, table = state["tokens"].long(), state["kv_len"].long(), state["table"]
    width = table.shape[1]
    free, n_free = state["free"], state["n_free"].long()

    def pages(n):
        return (n + ps - 1) // ps

    # what sequences drop goes on the stack of free pages
    left = (kv + tokens.clamp(max=0)).clamp(min=0)
    nth = torch.arange(width, device="cuda")[None]
    back = table[(nth >= pages(left)[:, None]) & (nth < pages(kv)[:, None])]
    free[n_free + torch.arange(back.numel(), device="cuda")] = back
    n_free = n_free + back.numel()
    # requests in their order; one that does not fit holds its place
    asks = (tokens > 0) & (kv + tokens <= width * ps)
    want = torch.where(asks, tokens, 0)
    need = pages(kv + want) - pages(kv)
    fits = asks & ((need == 0) | (need.cumsum(0) <= n_free)) & (want.cumsum(0) <= state["rows"])
    grown = left + torch.where(fits, want, 0)
    new = (nth >= pages(kv)[:, None]) & (nth < pages(grown)[:, None])
    taken = new.sum()
    at = n_free - new.flatten().long().cumsum(0).view_as(new)
    table.copy_(torch.where(new, free[torch.where(new, at, 0)], table))
    start = torch.cat([torch.zeros_like(kv[:1]), torch.where(fits, want, 0).cumsum(0)])
    row = torch.arange(state["rows"], device="cuda")
    seq = (torch.searchsorted(start, row, right=True) - 1).clamp(max=kv.numel() - 1)
    real = row < start[-1]
    pos = torch.where(real, grown[seq] - (start[seq + 1] - row), 0)
    slot = table[seq, pos // ps].long() * ps + pos % ps
    state["kv_out"].copy_(grown)
    state["n_free_out"].copy_(n_free - taken)
    state["start"].copy_(start)
    state["slots"].copy_(torch.where(real, slot, -1))
    state["positions"].copy_(torch.where(real, pos, -1))
    return _planned(state)


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    return x * cos + torch.cat([-hi, lo], -1) * sin


def _blocks(state, rows, kv):
    """The blocks of positions that the call's rows lie in: sequence, block, the
    packed row of each of its positions, and which are this call's and which older."""
    start, kv_len = state["start"].long(), state["kv_len"].long()
    first = kv_len - (start[1:] - start[:-1])
    count = torch.where(first < kv_len, (kv_len - 1) // BLOCK - first // BLOCK + 1, 0)
    total = sum((k - 1) // BLOCK - (k - r) // BLOCK + 1 for r, k in zip(rows, kv) if r)
    unit = torch.arange(total, device="cuda")
    seq = torch.searchsorted(count.cumsum(0), unit, right=True)
    block = first[seq] // BLOCK + unit - (count.cumsum(0) - count)[seq]
    pos = block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    new = (pos >= first[seq, None]) & (pos < kv_len[seq, None])
    at = (start[seq] - first[seq])[:, None] + pos
    return seq, block, torch.where(new, at, 0), torch.where(new, pos, 0), new, pos < first[seq, None]


def _plain_append(state):
    case = state["case"]
    h, hk, d, per = case["heads"], case["kv_heads"], case["dim"], case["page"] // BLOCK
    start, kv_len = state["start"].long(), state["kv_len"].long()
    n = state["q"].shape[0]
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = kv_len[seq] - (start[seq + 1] - row)
    state["out"].copy_(_rotate(state["q"].float().view(n, h, d), state["cos"][pos][:, None], state["sin"][pos][:, None]).view(n, h * d))
    seq, block, at, pos, new, old = _blocks(state, *_lengths(case))
    page, within = state["table"][seq, block // per].long(), block % per
    k = _rotate(state["k"].float().view(n, hk, d)[at], state["cos"][pos][:, :, None], state["sin"][pos][:, :, None])
    v = state["v"].float().view(n, hk, d)[at]
    _store(state, "k", page, within, k, new, old)
    _store(state, "v", page, within, v, new, old)
    return _appended(state)


def _store(state, name, page, within, x, new, old):
    """Rows x [blocks, BLOCK, hk, d] into the cache's blocks, beside the older rows
    in them, whose codes are rounded again where the block's scale grows."""
    x, new, old = x.transpose(1, 2), new[:, None, :, None], old[:, None, :, None]
    n_pages, hk, ps, d = state[name + "_pages"].shape
    pool = state[name + "_pages"].view(torch.uint8).view(n_pages, hk, ps // BLOCK, BLOCK, d)
    scales = state[name + "_scales"].view(torch.uint8)
    codes, was = pool[page, :, within], scales[page, :, within].int() - 127
    e = _exponent(torch.where(new, x, 0.0).abs().amax((2, 3)))
    e = torch.where(old.any(2)[..., 0], torch.maximum(e, was), e)
    again = codes.view(CODE).float() * _power((was - e).clamp(-127, 0))[..., None, None]
    put = torch.where(new, (x * _power(-e)[..., None, None]).to(CODE).view(torch.uint8), again.to(CODE).view(torch.uint8))
    pool[page, :, within] = torch.where(new | old, put, codes)
    scales[page, :, within] = (e + 127).to(torch.uint8)


def _plain_attention(state):
    case = state["case"]
    h, hk, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    grp = h // hk
    start, kv_len, table = state["start"].long(), state["kv_len"].long(), state["table"].long()
    rows = start[1:] - start[:-1]
    most = max(_lengths(case)[0])
    nth = torch.arange(most, device="cuda")
    real = nth[None] < rows[:, None]                                                  # [seqs, most]
    at = (start[:-1, None] + nth[None]).clamp(max=state["q"].shape[0] - 1)
    q = state["q"].float().view(-1, hk, grp, d)[at]                                   # [seqs, most, hk, grp, d]
    last = kv_len[:, None] - rows[:, None] + nth[None]                                # the rows' positions
    seqs, length = table.shape[0], table.shape[1] * ps
    seen = torch.arange(length, device="cuda")[None, None] <= last[:, :, None]        # [seqs, most, length]
    out = torch.zeros(seqs, most, hk, grp, d, device="cuda")

    def cached(name, i, step):
        codes = state[name + "_pages"].view(torch.uint8)[:, i:i + step][table].view(CODE).float()
        scales = state[name + "_scales"].view(torch.uint8)[:, i:i + step][table].view(SCALE).float()
        x = codes.view(*codes.shape[:3], ps // BLOCK, BLOCK, d).mul_(scales[..., None, None])
        return x.transpose(1, 2).reshape(seqs, -1, length, d)

    # as many KV heads at once as 4 GiB of scores and gathered rows hold
    step = max(1, (1 << 30) // (seqs * length * max(most * grp, 2 * d)))
    for i in range(0, hk, step):
        k, v = cached("k", i, step), cached("v", i, step)
        n = k.shape[1]
        s = torch.matmul(q[:, :, i:i + n].transpose(1, 2).reshape(seqs, n, most * grp, d), k.transpose(2, 3).contiguous())
        s = s.view(seqs, n, most, grp, length).mul_(state["scale"]).masked_fill_(~seen[:, None, :, None], -math.inf)
        s = s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(seqs, n, most * grp, length), v).view(seqs, n, most, grp, d)
        out[:, :, i:i + n] = torch.where(total > 0, o / total, 0.0).transpose(1, 2)
    state["out"].copy_(out.view(seqs, most, h * d)[real])
    return state["out"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _plain_plan(state) if kind == "plan" else _plain_append(state) if kind == "append" else _plain_attention(state)


# ---- the definition in 64 bits, one sequence after the other ----

def _exact_plan(case, state):
    ps = case["page"]
    tokens, kv = _lengths(case)
    table, free = state["table"].tolist(), state["free"].tolist()
    width, n_pages, rows = _plan_sizes(case)
    have = int(state["n_free"])
    start, slots, positions = [0], [], []
    for s, t in enumerate(tokens):
        if t < 0:
            end = max(0, kv[s] + t)
            for i in range(-(-end // ps), -(-kv[s] // ps)):
                free[have] = table[s][i]
                have += 1
            kv[s] = end
    asked_pages = asked_rows = 0
    top = have
    for s, t in enumerate(tokens):
        if t > 0 and kv[s] + t <= width * ps:
            a, b = -(-kv[s] // ps), -(-(kv[s] + t) // ps)
            asked_pages += b - a
            asked_rows += t
            if (a == b or asked_pages <= top) and asked_rows <= rows:
                for i in range(a, b):
                    have -= 1
                    table[s][i] = free[have]
                for j in range(kv[s], kv[s] + t):
                    slots.append(table[s][j // ps] * ps + j % ps)
                    positions.append(j)
                kv[s] += t
        start.append(len(slots))
    pad = [-1] * (rows - len(slots))

    def ints(a, dtype=torch.int32):
        return torch.tensor(a, dtype=dtype, device="cuda")

    return {"table": ints(table), "kv_out": ints(kv), "free": ints(free), "n_free_out": ints([have]),
            "start": ints(start), "slots": ints(slots + pad, torch.int64), "positions": ints(positions + pad)}


def _to_e4m3(y):
    """f64 values of at most 448 to e4m3's nearest, ties to even: steps of 2^-3 of the
    power of two below, of 2^-9 below 2^-6."""
    step = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4)
    return torch.round(y / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(case, state)
    rows, kv = _lengths(case)
    h, hk, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q = state["q"].double()
    n = q.shape[0]
    out = torch.zeros(n, h, d, dtype=torch.float64, device="cuda")
    at = 0
    if case["kind"] == "append":
        codes = {p: state[p + "_pages"].double() for p in "kv"}
        scales = {p: state[p + "_scales"].double() for p in "kv"}
        for s, (r, end) in enumerate(zip(rows, kv)):
            pos = torch.arange(end - r, end, device="cuda")
            c, sn = state["cos"].double()[pos, None, :d // 2], state["sin"].double()[pos, None, :d // 2]

            def turned(x, heads):
                z = x[at:at + r].double().reshape(r, heads, 2, d // 2)
                return torch.cat([z[:, :, 0] * c - z[:, :, 1] * sn, z[:, :, 1] * c + z[:, :, 0] * sn], -1)

            out[at:at + r] = turned(q, h)
            new = {"k": turned(state["k"], hk), "v": state["v"][at:at + r].double().reshape(r, hk, d)}
            first = (end - r) // BLOCK * BLOCK
            for b in range(first, end if r else first, BLOCK):
                lo, hi = max(b, end - r), min(b + BLOCK, end)
                page, i = int(state["table"][s, b // ps]), b % ps
                for p in "kv":
                    x = new[p][lo - end + r:hi - end + r].transpose(0, 1)  # [hk, rows, d]
                    amax = x.abs().amax((1, 2))
                    scale = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(min=-127))
                    scale = torch.where(amax > 448 * scale, 2 * scale, torch.where(amax <= 224 * scale, scale / 2, scale))
                    if lo > b:
                        was = scales[p][page, :, i // BLOCK]
                        scale = torch.maximum(scale, was)
                        older = codes[p][page, :, i:i + lo - b]
                        codes[p][page, :, i:i + lo - b] = _to_e4m3(older * (was / scale)[:, None, None])
                    codes[p][page, :, i + lo - b:i + hi - b] = _to_e4m3(x / scale[:, None, None])
                    scales[p][page, :, i // BLOCK] = scale
            at += r
        return {"out": out.view(n, h * d), "k_pages": codes["k"], "v_pages": codes["v"], "k_scales": scales["k"],
                "v_scales": scales["v"]}
    for s, (r, end) in enumerate(zip(rows, kv)):
        if r and end:
            page = state["table"][s, :-(-end // ps)].long()
            later = torch.arange(end, device="cuda")[None] > torch.arange(end - r, end, device="cuda")[:, None]

            def cached(name):
                unit = state[name + "_scales"].view(torch.uint8)[page].view(SCALE).double().repeat_interleave(BLOCK, 2)
                x = state[name + "_pages"].view(torch.uint8)[page].view(CODE).double() * unit[..., None]
                return x.permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :end]

            k, v = cached("k"), cached("v")
            for j in range(h):
                z = (q[at:at + r, j * d:(j + 1) * d] * state["scale"]) @ k[j * hk // h].t()
                z[later] = -math.inf
                out[at:at + r, j] = torch.softmax(z, -1) @ v[j * hk // h]
        at += r
    return out.view(n, h * d)
