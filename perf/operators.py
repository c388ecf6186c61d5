"""Performance cases of the paged KV cache operators: what a program that serves
a batch of sequences calls per layer between the QMatMuls.

  append    RoPE of the packed q and k rows, k and v appended to the cache's pages
  decode    attention of one new token per sequence over the pages
  prefill   causal attention of packed prompt rows (or of a chunk of a prompt
            whose earlier part is cached already) over the pages

Layer shapes are a 7B decoder's (32 heads of 128, as bench.py runs) and generic
grouped-head ones; ``draw`` covers the same kinds over smaller, odd and ragged
sizes.  q, k and v are N(0, 1) rows as a norm and a projection leave them, the
cache holds rows of the same kind, and the pages of a sequence are scattered
over the pool as an allocator leaves them after some hours.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # False: the plain forms; True: the package's kernels

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ----
# n_seqs sequences; their lengths before the call are spread between past_lo and
# past_hi and their new rows between new_lo and new_hi (over the logarithm, by
# `mix`); every `idle`-th slot of the batch holds no sequence (0: none).

def listed():
    seven = {"heads": 32, "kv_heads": 32, "dim": 128, "act": "f32", "cache": "f16", "page": 16, "mix": 1, "idle": 0}
    grouped = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "mix": 2, "idle": 0}
    one = {"new_lo": 1, "new_hi": 1}
    return [
        # one token of one sequence of a 7B decoder: the smallest append
        dict(seven, name="append_token", kind="append", seqs=1, past_lo=511, past_hi=511, **one),
        # one token each of a large batch, bf16 activations
        dict(grouped, name="append_batch", kind="append", act="bf16", cache="bf16", seqs=256, past_lo=8,
             past_hi=1000, **one),
        # a packed batch of ragged prompts, f32 projections as frq_qmatmul writes them
        dict(grouped, name="append_prompts", kind="append", act="f32", cache="f16", seqs=19, past_lo=0, past_hi=0,
             new_lo=33, new_hi=2048),
        # one token of a 7B decoder after a conversation of 700: the smallest attention
        dict(seven, name="decode_token", kind="decode", seqs=1, past_lo=700, past_hi=700, **one),
        # one sequence with a very long context: the split over the length
        dict(grouped, name="decode_long", kind="decode", act="f16", cache="f16", seqs=1, past_lo=131070,
             past_hi=131070, **one),
        # a serving batch of mixed lengths with idle slots
        dict(grouped, name="decode_ragged", kind="decode", act="bf16", cache="bf16", seqs=64, past_lo=16,
             past_hi=8191, idle=13, **one),
        # f32 activations (frq_qmatmul's output) over an f16 cache, eight query heads a KV head
        dict(grouped, name="decode_f32", kind="decode", kv_heads=4, act="f32", cache="f16", seqs=16, past_lo=1500,
             past_hi=4095, mix=3, **one),
        # many sequences of a model with heads of 64, larger pages
        dict(grouped, name="decode_dim64", kind="decode", heads=64, dim=64, act="f16", cache="f16", seqs=128,
             past_lo=200, past_hi=2048, page=64, mix=4, **one),
        # one short prompt, where the wait counts
        dict(grouped, name="prefill_short", kind="prefill", act="f16", cache="f16", seqs=1, past_lo=0, past_hi=0,
             new_lo=131, new_hi=131),
        # a packed batch of ragged prompts
        dict(grouped, name="prefill_ragged", kind="prefill", act="bf16", cache="bf16", seqs=17, past_lo=0, past_hi=0,
             new_lo=64, new_hi=2048, mix=5),
        # one long prompt
        dict(grouped, name="prefill_long", kind="prefill", act="bf16", cache="bf16", seqs=1, past_lo=0, past_hi=0,
             new_lo=16384, new_hi=16384),
        # a chunk of a 7B decoder's prompt after its cached part, f32 activations
        dict(seven, name="prefill_chunk_f32", kind="prefill", seqs=2, past_lo=3500, past_hi=7000, new_lo=300,
             new_hi=512),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (16, 2), (8, 1), (28, 4), (40, 8), (64, 8), (20, 1)])
    act, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([128, 128, 64]), "act": act,
            "cache": cache, "page": rng.choice([16, 16, 32, 64, 256]), "mix": rng.randint(1, 10 ** 6),
            "idle": rng.choice([0, 0, 3, 7])}
    per_token = kv_heads * case["dim"] * 4
    if kind == "decode":
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, min(131072, (400 << 20) // (per_token * seqs))))
        return dict(case, seqs=seqs, past_lo=rng.randint(0, hi), past_hi=hi, new_lo=1, new_hi=1)
    if kind == "append":
        seqs = _log(rng, 1, 256)
        new = rng.choice([1, _log(rng, 1, max(1, 16384 // seqs))])
        past = _log(rng, 1, 512)
        return dict(case, seqs=seqs, past_lo=rng.randint(0, past), past_hi=past, new_lo=_log(rng, 1, new), new_hi=new)
    seqs = _log(rng, 1, 32)
    # the plain form's scores: seqs * rows * length * heads values at most
    most = 16384 * 8192 // seqs * 32 // heads
    new = _log(rng, 1, min(8192, math.isqrt(most)))
    past = rng.choice([0, _log(rng, 1, max(1, min(16384, most // new - new)))])
    return dict(case, seqs=seqs, past_lo=rng.randint(0, past), past_hi=past, new_lo=_log(rng, 1, new), new_hi=new)


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return lo if lo == hi else min(hi, max(lo, _log(rng, max(1, lo), hi)))


def _lengths(case):
    """(rows, kv_len) of every slot: host lists, by the case alone."""
    rng = random.Random(case["mix"])
    rows, kv = [], []
    for s in range(case["seqs"]):
        new, past = _spread(rng, case["new_lo"], case["new_hi"]), _spread(rng, case["past_lo"], case["past_hi"])
        idle = case["idle"] and s % case["idle"] == case["idle"] - 1
        if case["kind"] == "decode":  # one row a slot, also where it is idle
            rows.append(1)
            kv.append(0 if idle else past + new)
        else:
            rows.append(0 if idle else new)
            kv.append(0 if idle else past + new)
    if not sum(rows):
        rows[0], kv[0] = 1, 1
    return rows, kv


def work(case):
    rows, kv = _lengths(case)
    a, c, d = SIZE[case["act"]], SIZE[case["cache"]], case["dim"]
    h, hk = case["heads"], case["kv_heads"]
    n = sum(rows)
    if case["kind"] == "append":
        positions = set()
        for r, k in zip(rows, kv):
            positions.update(range(k - r, k))
        # q read and written, k and v read and their cache rows written, the tables' rows
        return {"bytes": n * (2 * h * d * a + 2 * hk * d * (a + c)) + len(positions) * 2 * d * 4,
                "flops": 3 * n * (h + hk) * d}
    # K and V of every sequence once, q and out once; two products per visible pair
    pairs = sum(r * k - r * (r - 1) // 2 for r, k in zip(rows, kv) if k)
    return {"bytes": 2 * sum(kv) * hk * d * c + 2 * n * h * d * a, "flops": 4 * h * d * pairs}


# ---- inputs ----

def prepare(case, seed):
    if own:
        _one_stream()
    g = torch.Generator("cuda").manual_seed(seed)
    rng = random.Random(seed)
    rows, kv = _lengths(case)
    h, hk, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    act, cache = TORCH[case["act"]], TORCH[case["cache"]]
    need = [-(-k // ps) for k in kv]
    width, n_pages = max(max(need), 1), sum(need) + 7
    order = list(range(n_pages))
    rng.shuffle(order)
    table = torch.zeros(len(kv), width, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    n = start[-1]

    def normal(*shape, dtype=act):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    shape = (n_pages, hk, ps, d)
    state = {"case": case, "scale": 1.0 / math.sqrt(d), "table": table.cuda(), "max_kv_len": max(kv),
             "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda"),
             "start": torch.tensor(start, dtype=torch.int32, device="cuda")}
    if case["kind"] == "append":
        # q, k and v as one projection leaves them: a row of each token, one after the other
        qkv = normal(n, (h + 2 * hk) * d)
        state.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + hk) * d], v=qkv[:, (h + hk) * d:],
                     k_pages=torch.zeros(shape, dtype=cache, device="cuda"),
                     v_pages=torch.zeros(shape, dtype=cache, device="cuda"), out=torch.empty(n, h * d, dtype=act, device="cuda"))
        angle = torch.arange(max(kv), dtype=torch.float64)[:, None] * \
            10000.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64) / d)
        state.update(cos=torch.cat([angle.cos()] * 2, 1).float().cuda(), sin=torch.cat([angle.sin()] * 2, 1).float().cuda())
    else:
        state.update(q=normal(n, h * d), k_pages=normal(*shape, dtype=cache), v_pages=normal(*shape, dtype=cache),
                     out=torch.empty(n, h * d, dtype=act, device="cuda"))
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
    code = {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}
    n_pages = state["k_pages"].shape[0]
    cache = F.PagedKvCache(_device, n_pages, case["page"], case["kv_heads"], case["dim"], code[case["cache"]],
                           k=state["k_pages"].data_ptr(), v=state["v_pages"].data_ptr())
    batch = F.PagedBatch(state["table"].data_ptr(), state["kv_len"].data_ptr(), case["seqs"],
                         state["table"].shape[1], state["q"].shape[0],
                         row_start=None if case["kind"] == "decode" else state["start"].data_ptr(),
                         max_kv_len=state["max_kv_len"])
    work = None
    if case["kind"] != "append":
        work = _device.alloc((max(1, F.paged_attention_workspace(cache, batch, case["heads"])),), "uint8")
    return F, cache, batch, code[case["act"]], work


def _run_own(state):
    F, cache, batch, act, work = state["handle"]
    case = state["case"]
    q, out = state["q"], state["out"]
    if case["kind"] == "append":
        F.paged_append(cache, batch, act, case["heads"], q.data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(),
                       out.data_ptr(), ldq=q.stride(0), ldk=state["k"].stride(0), ldv=state["v"].stride(0),
                       rope_cos=state["cos"].data_ptr(), rope_sin=state["sin"].data_ptr(), rope_rows=state["cos"].shape[0])
        return out, state["k_pages"], state["v_pages"]
    attend = F.paged_attention_decode if case["kind"] == "decode" else F.paged_attention_prefill
    attend(cache, batch, act, case["heads"], q.data_ptr(), out.data_ptr(), state["scale"], work)
    return out


# ---- the plain forms ----

def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    return x * cos + torch.cat([-hi, lo], -1) * sin


def _plain_append(state):
    case = state["case"]
    h, hk, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    start, kv_len = state["start"].long(), state["kv_len"].long()
    n = state["q"].shape[0]
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = kv_len[seq] - (start[seq + 1] - row)
    cos, sin = state["cos"][pos][:, None], state["sin"][pos][:, None]
    q = _rotate(state["q"].float().view(n, h, d), cos, sin)
    k = _rotate(state["k"].float().view(n, hk, d), cos, sin)
    page, slot = state["table"][seq, pos // ps].long(), pos % ps
    state["k_pages"][page, :, slot] = k.to(state["k_pages"].dtype)
    state["v_pages"][page, :, slot] = state["v"].float().view(n, hk, d).to(state["v_pages"].dtype)
    state["out"].copy_(q.view(n, h * d))
    return state["out"], state["k_pages"], state["v_pages"]


def _plain_attention(state):
    case = state["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    grp = h // hk
    start, kv_len, table = state["start"].long(), state["kv_len"].long(), state["table"].long()
    rows = start[1:] - start[:-1]
    most = max(_lengths(case)[0])
    nth = torch.arange(most, device="cuda")
    real = nth[None] < rows[:, None]                                                  # [seqs, most]
    at = (start[:-1, None] + nth[None]).clamp(max=state["q"].shape[0] - 1)
    q = state["q"].float().view(-1, hk, grp, d)[at]                                   # [seqs, most, hk, grp, d]
    last = kv_len[:, None] - rows[:, None] + nth[None]                                # the rows' positions
    seqs, length = table.shape[0], table.shape[1] * case["page"]
    seen = torch.arange(length, device="cuda")[None, None] <= last[:, :, None]        # [seqs, most, length]
    out = torch.zeros(seqs, most, hk, grp, d, device="cuda")
    # as many KV heads at once as 4 GiB of scores and gathered rows hold
    step = max(1, (1 << 30) // (seqs * length * max(most * grp, 2 * d)))
    for i in range(0, hk, step):
        k, v = (state[p][:, i:i + step][table].transpose(1, 2).reshape(seqs, -1, length, d).float()
                for p in ("k_pages", "v_pages"))
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
    return _plain_append(state) if state["case"]["kind"] == "append" else _plain_attention(state)


# ---- the definition in 64 bits, one sequence after the other ----

def exact(case, seed):
    state = prepare(case, seed)
    rows, kv = _lengths(case)
    h, hk, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q = state["q"].double()
    n = q.shape[0]
    out = torch.zeros(n, h, d, dtype=torch.float64, device="cuda")
    at = 0
    if case["kind"] == "append":
        pages = [torch.zeros(state[p].shape, dtype=torch.float64, device="cuda") for p in ("k_pages", "v_pages")]
        for s, (r, end) in enumerate(zip(rows, kv)):
            pos = torch.arange(end - r, end, device="cuda")
            c, sn = state["cos"].double()[pos, None, :d // 2], state["sin"].double()[pos, None, :d // 2]

            def turned(x, heads):
                z = x[at:at + r].double().reshape(r, heads, 2, d // 2)
                return torch.cat([z[:, :, 0] * c - z[:, :, 1] * sn, z[:, :, 1] * c + z[:, :, 0] * sn], -1)

            out[at:at + r] = turned(q, h)
            page, slot = state["table"][s].long()[pos // ps], pos % ps
            pages[0][page, :, slot] = turned(state["k"], hk)
            pages[1][page, :, slot] = state["v"][at:at + r].double().reshape(r, hk, d)
            at += r
        return out.view(n, h * d), pages[0], pages[1]
    for s, (r, end) in enumerate(zip(rows, kv)):
        if r and end:
            page = state["table"][s, :-(-end // ps)].long()
            later = torch.arange(end, device="cuda")[None] > torch.arange(end - r, end, device="cuda")[:, None]
            k, v = (state[p][page].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :end].double() for p in ("k_pages", "v_pages"))
            for j in range(h):
                z = (q[at:at + r, j * d:(j + 1) * d] * state["scale"]) @ k[j * hk // h].t()
                z[later] = -math.inf
                out[at:at + r, j] = torch.softmax(z, -1) @ v[j * hk // h]
        at += r
    return out.view(n, h * d)
