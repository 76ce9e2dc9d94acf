"""The operators of one continuous-batching step over the paged fp8 cache, in their plain form and as this framework
offers them.

- listed()            named cases: the smallest calls, ordinary ones, the largest
- draw(rng)           one more case of the same ranges
- prepare(case, seed) what a serving program holds before the call: its inputs, cache, block tables and handles
- run(state)          one pass; with `own` false in elementary torch operations, else through nanochat_amd
- work(case)          bytes and flops one pass cannot do without
- exact(case, seed)   run's outputs from the definitions, in float64

Kinds of case, in the order a step uses them:

  pages   block tables and slot maps from the requests' lengths: the step's tokens get their pages, positions and cache
          slots (paging.BlockTables.extend), and a rollback gives the pages back (BlockTables.trim)
  append  QK norm, RoPE and the fp8 store of packed rows by slot map (attention.qk_norm_rope_append_packed)
  attend  attention of packed rows, any number of new tokens a sequence, over the paged cache (attention.packed_attention)
  sample  a token a row from its logits, by temperature, top-k, top-p and min-p from given random numbers
          (sampling.sample_tokens)
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
D, PAGE = 128, 16
EPS = torch.finfo(torch.float32).eps
FP8_MAX = 448.0


def listed():
    return [
        # A decoding step's bookkeeping: 128 slots, one new token each, at lengths of their own up to 2,560.
        dict(name="pages_step", kind="pages", slots=128, idle=0.1, new_lo=1, new_hi=1, ctx=2560, rows=128, short=False),
        # Prompt chunks beside decoding: 512 slots take 1 to 64 tokens each, and the pool cannot hold them all.
        dict(name="pages_prompts", kind="pages", slots=512, idle=0.2, new_lo=1, new_hi=64, ctx=8192, rows=16384,
             short=True),
        # The new rows of a decoding batch: 64 sequences, grouped-query heads.
        dict(name="append_step", kind="append", seqs=64, new_lo=1, new_hi=1, ctx=8192, q_heads=16, kv_heads=4),
        # Prompt chunks of eight requests, no round length, at positions of no round offset: 4,096 rows at most.
        dict(name="append_chunks", kind="append", seqs=8, new_lo=257, new_hi=512, ctx=3584, q_heads=16, kv_heads=4),
        # One user, five draft tokens to verify, the small model's 6 heads, 1,024 cached tokens. Latency is all.
        dict(name="attend_verify_one", kind="attend", seqs=1, new_lo=5, new_hi=5, few=0, ctx_lo=1024, ctx=1024,
             q_heads=6, kv_heads=6, window=-1),
        # A full batch with four draft tokens a sequence at its longest context.
        dict(name="attend_verify_8k", kind="attend", seqs=64, new_lo=4, new_hi=4, few=0, ctx_lo=8192, ctx=8192,
             q_heads=16, kv_heads=4, window=-1),
        # A server in mid-flight: 60 sequences decode one token, four take prompt chunks, each at a length of its own.
        dict(name="attend_mixed", kind="attend", seqs=64, new_lo=200, new_hi=700, few=60, ctx_lo=512, ctx=8192,
             q_heads=16, kv_heads=4, window=-1),
        # Chunked prefill: 512-token chunks of eight prompts onto 3,584 cached tokens each.
        dict(name="attend_chunks", kind="attend", seqs=8, new_lo=512, new_hi=512, few=0, ctx_lo=3584, ctx=3584,
             q_heads=16, kv_heads=4, window=-1),
        # New prompts of mixed lengths, nothing cached, on a windowed layer of the 13-head model.
        dict(name="attend_prompts", kind="attend", seqs=7, new_lo=130, new_hi=2048, few=0, ctx_lo=0, ctx=0, q_heads=13,
             kv_heads=13, window=700),
        # One user's next token, by temperature and a nucleus, of the 65,536-token vocabulary.
        dict(name="sample_one", kind="sample", rows=1, vocab=65536, dtype="float32", temp=0.8, top_k=0, top_p=0.95,
             min_p=0.0, greedy=0.0, spread=2.5, mask=False),
        # A full batch, every row with settings of its own, a quarter of them greedy.
        dict(name="sample_batch", kind="sample", rows=128, vocab=65536, dtype="float32", temp=1.0, top_k=50, top_p=0.9,
             min_p=0.05, greedy=0.25, spread=2.5, mask=False),
        # Near-flat bf16 logits under allowed-token masks, an odd number of rows, no top-k to narrow them.
        dict(name="sample_flat", kind="sample", rows=333, vocab=32768, dtype="bfloat16", temp=1.3, top_k=0, top_p=0.98,
             min_p=0.0, greedy=0.0, spread=0.5, mask=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_pages(rng):
    slots, ctx, hi = _log_int(rng, 1, 1024), _log_int(rng, 16, 16384), _log_int(rng, 1, 512)
    while slots * hi > 32768:
        hi = max(1, hi // 2)
    return dict(kind="pages", slots=slots, idle=rng.choice([0.0, 0.1, 0.5]), new_lo=rng.choice([0, 1, hi]), new_hi=hi,
                ctx=ctx, rows=max(1, slots * hi - rng.randint(0, max(1, slots * hi // 3))), short=rng.random() < 0.3)


def _draw_append(rng):
    hq, hkv = rng.choice([(6, 6), (10, 10), (13, 13), (16, 4), (8, 1), (12, 4)])
    seqs, hi, ctx = _log_int(rng, 1, 128), _log_int(rng, 1, 2048), rng.choice([0, _log_int(rng, 1, 8192)])
    while seqs * hi > 8192:
        hi = max(1, hi // 2)
    return dict(kind="append", seqs=seqs, new_lo=rng.choice([1, hi]), new_hi=hi, ctx=ctx, q_heads=hq, kv_heads=hkv)


def _draw_attend(rng):
    hq, hkv = rng.choice([(6, 6), (10, 10), (13, 13), (16, 4), (8, 1), (12, 4), (16, 1)])
    seqs, hi, ctx = _log_int(rng, 1, 64), _log_int(rng, 1, 2000), rng.choice([0, _log_int(rng, 16, 8192)])
    few = rng.choice([0, 0, seqs // 2, seqs])
    cost = lambda: ((seqs - few) * hi + few) * hq * (ctx + hi) + seqs * (ctx + hi) * hkv * 16  # noqa: E731
    while cost() > 8 * 512 * 16 * 4096:
        if hi > 1:
            hi = max(1, hi * 3 // 4)
        ctx = ctx * 7 // 8
    return dict(kind="attend", seqs=seqs, new_lo=rng.choice([1, hi]), new_hi=hi, few=few,
                ctx_lo=rng.choice([ctx, ctx // 16]), ctx=ctx, q_heads=hq, kv_heads=hkv,
                window=rng.choice([-1, -1, 300, 1024]))


def _draw_sample(rng):
    rows, vocab = _log_int(rng, 1, 512), rng.choice([_log_int(rng, 64, 100000), 32768, 65536])
    while rows * vocab > 128 * 65536:
        rows = max(1, rows // 2)
    return dict(kind="sample", rows=rows, vocab=vocab, dtype=rng.choice(["float32", "float32", "bfloat16"]),
                temp=rng.choice([0.6, 1.0, 2.0]), top_k=rng.choice([0, 0, 1, 20, 300]),
                top_p=rng.choice([1.0, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.02]),
                greedy=rng.choice([0.0, 0.3]), spread=rng.choice([0.5, 2.5, 5.0]), mask=rng.random() < 0.3)


def draw(rng):
    return rng.choice([_draw_pages, _draw_append, _draw_attend, _draw_sample])(rng)


# --- lengths: those of a case are its own, so that work() knows them

def _requests(case):
    """(new tokens, cached tokens) of every sequence of an append or attend case."""
    rng = random.Random(f"{case['seqs']} {case['new_lo']} {case['new_hi']} {case['ctx']}")
    few, lo = case.get("few", 0), case.get("ctx_lo", 0)
    new = [1 if b < few else rng.randint(min(case["new_lo"], case["new_hi"]), case["new_hi"])
           for b in range(case["seqs"])]
    ctx = [rng.randint(min(lo, case["ctx"]), case["ctx"]) for _ in range(case["seqs"])]
    order = list(range(case["seqs"]))
    rng.shuffle(order)
    return [new[b] for b in order], ctx


def _slots(case):
    """(new tokens, cached tokens) of every slot of a pages case, and its pool: pages in use and free."""
    rng = random.Random(f"{case['slots']} {case['new_hi']} {case['ctx']} {case['rows']}")
    ctx = [0 if rng.random() < case["idle"] else rng.randint(1, case["ctx"]) for _ in range(case["slots"])]
    new = [0 if c == 0 and rng.random() < 0.5 else rng.randint(min(case["new_lo"], case["new_hi"]), case["new_hi"])
           for c in ctx]
    used = sum(_pages(c) for c in ctx)
    need = sum(_pages(c + n) - _pages(c) for c, n in zip(ctx, new))
    free = max(1, need * 7 // 8) if case["short"] else need + 64
    return new, ctx, used, free


def _pages(length):
    return -(-length // PAGE)


# --- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _k_layout(x):
    """[.., 16 slots, 128] -> a K page's bytes [.., 2048]: byte h 1024 + (g 16 + slot) 16 + j holds dim 32 g + 16 h + j."""
    return x.unflatten(-1, (4, 2, 16)).permute(*range(x.dim() - 2), -2, -3, -4, -1).flatten(-4)


def _v_layout(x):
    """[.., 16 slots, 128] -> a V page's bytes [.., 2048]: byte (t / 4) 1024 + ((slot / 4) 16 + r) 16 + (t % 4) 4 +
    slot % 4 holds dim 16 t + r."""
    x = x.unflatten(-1, (2, 4, 16)).unflatten(-4, (4, 4))      # .., slot / 4, slot % 4, t / 4, t % 4, r
    return x.permute(*range(x.dim() - 5), -3, -5, -1, -2, -4).flatten(-5)


def _k_rows(pages):
    """K page bytes [.., 2048] -> [.., 16 slots, 128]."""
    x = pages.unflatten(-1, (2, 4, 16, 16))                    # h, g, slot, j
    return x.permute(*range(x.dim() - 4), -2, -3, -4, -1).flatten(-3)


def _v_rows(pages):
    """V page bytes [.., 2048] -> [.., 16 slots, 128]."""
    x = pages.unflatten(-1, (2, 4, 16, 4, 4))                  # t / 4, slot / 4, r, t % 4, slot % 4
    return x.permute(*range(x.dim() - 5), -4, -1, -5, -2, -3).flatten(-5, -4).flatten(-3)


def _filled_cache(gen, num_pages, heads):
    """A pool whose every slot holds a token: e4m3 codes in the pages' layout, one scale a (token, head)."""
    codes, scales = [], []
    for layout in (_k_layout, _v_layout):
        x = torch.randn(num_pages, heads, PAGE, D, generator=gen, device=DEVICE)
        amax = x.abs().amax(-1)
        scales.append(amax / FP8_MAX)
        codes.append(layout((x * (FP8_MAX / amax).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)))
    return dict(k_pages=codes[0].contiguous(), v_pages=codes[1].contiguous(), kv_scale=torch.stack(scales, 2))


def _cache_handle(cache):
    from nanochat_amd.kv_cache import PagedKVCache

    handle = PagedKVCache(cache["k_pages"].size(0), cache["k_pages"].size(1), DEVICE)
    for name in ("k_pages", "v_pages", "kv_scale"):
        getattr(handle, name).copy_(cache[name])
    return handle


def _random_table(gen, lengths):
    """A block table of scattered pages for sequences of these lengths, and the pages of the pool."""
    counts = [_pages(n) for n in lengths]
    perm = torch.randperm(sum(counts) + 1, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, perm.numel()


def _rotary(length, theta=1_000_000.0):
    freq = theta ** -(torch.arange(0, D, 2, dtype=torch.float64, device=DEVICE) / D)
    angle = torch.arange(length, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _prepare_pages(case, gen):
    new, ctx, used, free = _slots(case)
    num_pages = used + free
    perm = torch.randperm(num_pages, generator=gen, device=DEVICE).to(torch.int32)
    max_pages = _pages(max(c + n for c, n in zip(ctx, new))) + 1
    table = torch.full((case["slots"], max_pages), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, c in enumerate(ctx):
        table[b, :_pages(c)] = perm[at:at + _pages(c)]
        at += _pages(c)
    state = dict(case=case, new=_int32(new), keep=_int32(ctx), table=table, lengths=_int32(ctx),
                 free_pages=torch.cat([perm[used:], perm[:used]]), free_count=_int32([free]))
    if own:
        from nanochat_amd.paging import BlockTables

        state["tables"] = BlockTables(case["slots"], max_pages, num_pages, DEVICE)
        for name in ("table", "lengths", "free_pages", "free_count"):
            getattr(state["tables"], name).copy_(state[name])
    return state


def _prepare_append(case, gen):
    new, ctx = _requests(case)
    lengths = [n + c for n, c in zip(new, ctx)]
    table, num_pages = _random_table(gen, lengths)
    hq, hkv = case["q_heads"], case["kv_heads"]
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), torch.tensor(new, device=DEVICE))
    positions = torch.cat([torch.arange(c, c + n, device=DEVICE) for n, c in zip(new, ctx)])
    slot_map = table[seq, positions // PAGE] * PAGE + (positions % PAGE).to(torch.int32)
    cos, sin = _rotary(max(lengths))
    state = dict(case=case, qkv=_randn(gen, seq.numel(), (hq + 2 * hkv) * D, scale=1.5), cos=cos, sin=sin,
                 q_gain=1 + 0.1 * _randn(gen, D, dtype=torch.float32), k_gain=1 + 0.1 * _randn(gen, D, dtype=torch.float32),
                 positions=positions.to(torch.int32), slot_map=slot_map, cache=_filled_cache(gen, num_pages, hkv))
    if own:
        state["handle"] = _cache_handle(state["cache"])
    return state


def _prepare_attend(case, gen):
    new, ctx = _requests(case)
    lengths = [n + c for n, c in zip(new, ctx)]
    table, num_pages = _random_table(gen, lengths)
    state = dict(case=case, q=_randn(gen, sum(new), case["q_heads"], D), table=table, seq_lens=_int32(lengths),
                 cu_seqlens=torch.cat([_int32([0]), _int32(new).cumsum(0).to(torch.int32)]), new=new, lengths=lengths,
                 cache=_filled_cache(gen, num_pages, case["kv_heads"]))
    if own:
        state["handle"] = _cache_handle(state["cache"])
    return state


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    logits = _randn(gen, rows, vocab, dtype=torch.float32, scale=case["spread"])
    # a few tokens stand out in a confident row, none in a flat one
    peaks = torch.randint(0, vocab, (rows, 8), generator=gen, device=DEVICE)
    logits.scatter_add_(1, peaks, _randn(gen, rows, 8, dtype=torch.float32, scale=case["spread"]).abs() * 1.5)
    logits = (15.0 * torch.tanh(logits / 15.0)).to(getattr(torch, case["dtype"]))
    u = torch.rand(rows, 6, generator=gen, device=DEVICE)
    state = dict(case=case, logits=logits, uniform=u[:, 0].contiguous(),
                 temperature=torch.where(u[:, 1] < case["greedy"], 0.0, case["temp"] * (0.75 + 0.5 * u[:, 2])),
                 top_k=(case["top_k"] * (0.5 + u[:, 3])).to(torch.int32),
                 top_p=(1.0 - (1.0 - case["top_p"]) * (0.5 + u[:, 4])), min_p=case["min_p"] * u[:, 5], mask=None)
    if case["mask"]:
        state["mask"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen, device=DEVICE,
                                      dtype=torch.int64).to(torch.int32)
    return state


def prepare(case, seed):
    return {"pages": _prepare_pages, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["kind"]](case, _generator(seed))


# --- pages: the plain form

def _pages_of(lengths):
    return (lengths + PAGE - 1) // PAGE


def _plain_extend(s):
    """Slots in order take pages while the pool has enough (a slot that needs none is not refused for pages), then rows
    while the step has enough; a slot asks all or nothing. The j-th page granted is the j-th from the free list's end."""
    rows, max_pages = s["case"]["rows"], s["table"].size(1)
    old, asked = s["lengths"].long(), s["new"].long().clamp(min=0)
    asked = torch.where(old + asked <= max_pages * PAGE, asked, 0)
    need = _pages_of(old + asked) - _pages_of(old)
    fits = (need == 0) | (need.cumsum(0) <= s["free_count"])
    asked = torch.where(fits, asked, 0)
    granted = torch.where(asked.cumsum(0) <= rows, asked, 0)
    need = _pages_of(old + granted) - _pages_of(old)
    first = need.cumsum(0) - need
    cu = torch.cat([granted.new_zeros(1), granted.cumsum(0)])
    row = torch.arange(rows, device=DEVICE)
    live = row < cu[-1]
    seq = torch.searchsorted(cu[1:], row, right=True).clamp(max=old.numel() - 1)
    positions = torch.where(live, old[seq] + row - cu[seq], -1)
    page = positions.clamp(min=0) // PAGE
    fresh = page - _pages_of(old)[seq]
    taken = s["free_pages"][(s["free_count"] - 1 - first[seq] - fresh.clamp(min=0)).clamp(min=0)]
    held = torch.where(live & (fresh >= 0), taken, s["table"][seq, page])
    slot_map = torch.where(live, held * PAGE + positions % PAGE, -1)
    starts = live & (fresh >= 0) & (positions % PAGE == 0)      # each granted page's first row writes its entry
    at = torch.where(starts, seq * max_pages + page, s["table"].numel())
    padded = torch.cat([s["table"].flatten(), s["table"].new_zeros(1)])
    s["table"].copy_(padded.index_copy(0, at, held)[:-1].view_as(s["table"]))
    s["lengths"].copy_(old + granted)
    s["free_count"].sub_(need.sum().to(torch.int32))
    return [t.to(torch.int32) for t in (cu, positions, slot_map, granted)]


def _plain_trim(s):
    """Slots fall back to keep (where it is shorter); the pages past it join the free list, the last one first."""
    old = s["lengths"].long()
    kept = torch.where((s["keep"] >= 0) & (s["keep"] < old), s["keep"].long(), old)
    page = torch.arange(s["table"].size(1), device=DEVICE)
    gone = (page >= _pages_of(kept)[:, None]) & (page < _pages_of(old)[:, None])
    j = gone.flatten().cumsum(0) - 1
    count = gone.sum()
    at = torch.where(gone.flatten(), s["free_count"] + count - 1 - j, s["free_pages"].numel())
    padded = torch.cat([s["free_pages"], s["free_pages"].new_zeros(1)])
    s["free_pages"].copy_(padded.index_copy(0, at, s["table"].flatten())[:-1])
    s["table"].copy_(torch.where(gone, -1, s["table"]))
    s["lengths"].copy_(kept)
    s["free_count"].add_(count.to(torch.int32))


# --- append: the plain form

def _norm_rope(x, gain, cos, sin):
    """RMS norm, gain and -theta rotation of rows [.., 128] in fp32, the squares summed pairwise (dims l and l + 64, then
    halves), rounded once to bf16: the order the cache's codes are defined by."""
    x1, x2 = x.float().chunk(2, -1)
    total = x1 * x1 + x2 * x2
    total = total[..., :32] + total[..., 32:]
    total = total[..., :16] + total[..., 16:]
    total = total[..., :8] + total[..., 8:]
    total = total[..., :4] + total[..., 4:]
    total = total[..., :2] + total[..., 2:]
    total = total[..., :1] + total[..., 1:]
    root = (total / 128.0 + EPS).double().sqrt().float()
    r = (1.0 / root.double()).float()
    n1, n2 = x1 * r * gain[:64], x2 * r * gain[64:]
    return torch.cat([n1 * cos + n2 * sin, n2 * cos - n1 * sin], -1).to(torch.bfloat16)


def _quantize(x):
    """bf16 rows [.., 128] -> (e4m3 codes as bytes, scales): the largest magnitude of a row becomes 448."""
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, (amax.double() / FP8_MAX).float(), 1.0)
    y = (x.double() / scale.double().unsqueeze(-1)).float().clamp(-FP8_MAX, FP8_MAX)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), scale


def _plain_append(s):
    hq, hkv, cache = s["case"]["q_heads"], s["case"]["kv_heads"], s["cache"]
    x = s["qkv"].unflatten(-1, (hq + 2 * hkv, D))
    at = s["positions"].long()
    cos, sin = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)
    q = _norm_rope(x[:, :hq], s["q_gain"], cos, sin)
    k, k_scale = _quantize(_norm_rope(x[:, hq:hq + hkv], s["k_gain"], cos, sin))
    v, v_scale = _quantize(x[:, hq + hkv:])
    page, slot = s["slot_map"].long() // PAGE, s["slot_map"].long() % PAGE
    kp = cache["k_pages"].unflatten(-1, (2, 4, 16, 16))
    kp[page, :, :, :, slot] = k.unflatten(-1, (4, 2, 16)).transpose(2, 3)
    vp = cache["v_pages"].unflatten(-1, (2, 4, 16, 4, 4))
    vp[page, :, :, slot // 4, :, :, slot % 4] = v.unflatten(-1, (2, 4, 16)).transpose(3, 4)
    cache["kv_scale"][page, :, 0, slot] = k_scale
    cache["kv_scale"][page, :, 1, slot] = v_scale
    return [q, cache["k_pages"].view(torch.float8_e4m3fn), cache["v_pages"].view(torch.float8_e4m3fn), cache["kv_scale"]]


# --- attend: the plain form

def _plain_attend(s):
    """Padded batches: the sequences of one new token, then the others."""
    case, table, cache = s["case"], s["table"], s["cache"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    out = torch.empty_like(s["q"])
    for group in ([b for b, n in enumerate(s["new"]) if n == 1], [b for b, n in enumerate(s["new"]) if n != 1]):
        if not group:
            continue
        seqs = torch.tensor(group, device=DEVICE)
        n, pages = max(s["new"][b] for b in group), _pages(max(s["lengths"][b] for b in group))
        held = table[seqs, :pages].clamp(min=0).long()
        scale = cache["kv_scale"][held].unsqueeze(-1)                     # g, pages, Hkv, 2, 16, 1
        k = _k_rows(cache["k_pages"][held].view(torch.float8_e4m3fn).float()) * scale[:, :, :, 0]
        v = _v_rows(cache["v_pages"][held].view(torch.float8_e4m3fn).float()) * scale[:, :, :, 1]
        k, v = (t.transpose(1, 2).flatten(2, 3) for t in (k, v))          # g, Hkv, keys, 128
        first, count = s["cu_seqlens"][seqs].long(), s["cu_seqlens"][seqs + 1].long() - s["cu_seqlens"][seqs].long()
        step = torch.arange(n, device=DEVICE)
        live = step < count[:, None]
        rows = torch.where(live, first[:, None] + step, 0)
        position = (s["seq_lens"][seqs].long() - count)[:, None] + step   # g, n
        q = s["q"][rows].float().unflatten(2, (hkv, hq // hkv)).transpose(1, 2).flatten(2, 3)
        scores = q @ k.transpose(-1, -2) * D ** -0.5                      # g, Hkv, n G, keys
        key = torch.arange(k.size(2), device=DEVICE)
        seen = key <= position[..., None]
        if case["window"] >= 0:
            seen &= key >= position[..., None] - case["window"]
        seen = seen.repeat_interleave(hq // hkv, 1).unsqueeze(1)
        scores.masked_fill_(~seen, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        o = o.unflatten(2, (n, hq // hkv)).transpose(1, 2).flatten(2, 3).to(torch.bfloat16)
        out[rows[live]] = o[live]
    return out


# --- sample: the plain form

def _plain_sample(s):
    """Weights exp((z - max) / T) in float64; the top-k rows (the lower index first among equals), the tokens with less
    than top_p of the weight strictly above them, those of at least min_p times the largest; then the first token, in
    index order, whose running weight passes the uniform number's share. Temperature 0: the largest logit."""
    z = s["logits"].double()
    if s["mask"] is not None:
        word = torch.arange(z.size(1), device=DEVICE)
        z = z.masked_fill((s["mask"][:, word // 32] >> (word % 32).to(torch.int32) & 1) == 0, -math.inf)
    top, greedy = z.max(-1, keepdim=True)
    temperature = s["temperature"].double().unsqueeze(1)
    e = torch.exp((z - top) / torch.where(temperature > 0, temperature, 1.0))
    e = torch.where(z == -math.inf, 0.0, e)
    value, order = torch.sort(z, dim=-1, descending=True, stable=True)
    rank = torch.arange(z.size(1), device=DEVICE)
    k = s["top_k"].long().unsqueeze(1)
    sorted_e = torch.where((k <= 0) | (rank < k), e.gather(1, order), 0.0)
    running = sorted_e.cumsum(-1)
    # the weight strictly above a token: the running weight before the first of its equals
    starts = torch.cat([torch.ones_like(value[:, :1], dtype=torch.bool), value[:, 1:] != value[:, :-1]], 1)
    above = torch.where(starts, running - sorted_e, 0.0).cummax(-1).values
    top_p = s["top_p"].double().unsqueeze(1)
    inside = (above < top_p * running[:, -1:]) | (top_p >= 1) | (value == top)
    kept = torch.where(inside & (sorted_e >= s["min_p"].double().unsqueeze(1)), sorted_e, 0.0)
    share = torch.zeros_like(e).scatter(1, order, kept).cumsum(-1)
    target = s["uniform"].double().unsqueeze(1) * share[:, -1:]
    token = torch.searchsorted(share, target, right=True).squeeze(1).clamp(max=z.size(1) - 1)
    token = torch.where(s["temperature"] > 0, token, greedy.squeeze(1))
    return torch.where(top.squeeze(1) > -math.inf, token, -1).to(torch.int32)


# --- one pass

def _own_pages(s):
    maps = s["tables"].extend(s["new"], s["case"]["rows"])
    s["tables"].trim(s["keep"])
    t = s["tables"]
    return [maps.cu_seqlens, maps.positions, maps.slot_map, maps.granted, t.table, t.lengths, t.free_pages, t.free_count]


def _own_append(s):
    from nanochat_amd.attention import qk_norm_rope_append_packed

    h = s["handle"]
    q = qk_norm_rope_append_packed(s["qkv"], s["case"]["q_heads"], h, s["positions"], s["slot_map"], s["q_gain"],
                                   s["k_gain"], s["cos"], s["sin"])
    return [q, h.k_pages.view(torch.float8_e4m3fn), h.v_pages.view(torch.float8_e4m3fn), h.kv_scale]


def _own_attend(s):
    from nanochat_amd.attention import packed_attention

    return packed_attention(s["q"], s["handle"], s["table"], s["cu_seqlens"], s["seq_lens"], max(s["lengths"]),
                            window=s["case"]["window"])


def _own_sample(s):
    from nanochat_amd.sampling import sample_tokens

    return sample_tokens(s["logits"], s["uniform"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                         min_p=s["min_p"], mask=s["mask"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"pages": _own_pages, "append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](state)
    if kind == "pages":
        maps = _plain_extend(state)
        _plain_trim(state)
        return [*maps, *(state[name] for name in ("table", "lengths", "free_pages", "free_count"))]
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[kind](state)


# --- what a pass cannot do without

def _seen_keys(n, c, window):
    """Query-key products of a sequence's n new rows on c cached tokens, and the keys its rows see between them."""
    if window < 0:
        return n * c + n * (n + 1) // 2, c + n
    return sum(min(c + t, window) + 1 for t in range(n)), c + n - max(c - window, 0)


def work(case):
    if case["kind"] == "pages":
        new, ctx, _, free = _slots(case)
        granted = min(case["rows"], sum(new))
        pages = sum(_pages(c + n) - _pages(c) for c, n in zip(ctx, new))
        # lengths and requests in, cu, grants and lengths out, twice; a row's position and slot; a page's entry and place
        return {"bytes": 4.0 * (7 * case["slots"] + 2 * case["rows"] + 6 * min(pages, free)), "flops": 8.0 * granted}
    if case["kind"] == "sample":
        size = case["rows"] * case["vocab"]
        return {"bytes": size * (4.0 if case["dtype"] == "float32" else 2.0) + (size / 8 if case["mask"] else 0) +
                24.0 * case["rows"], "flops": 4.0 * size}
    new, ctx = _requests(case)
    rows, hq, hkv = sum(new), case["q_heads"], case["kv_heads"]
    if case["kind"] == "append":
        places = max(n + c for n, c in zip(new, ctx))
        return {"bytes": 256.0 * rows * (2 * hq + 2 * hkv) + 264.0 * rows * hkv + 8.0 * rows +
                512.0 * min(rows, places) + 1024, "flops": 128.0 * rows * (8 * hq + 11 * hkv)}
    pairs, keys = (sum(t) for t in zip(*(_seen_keys(n, c, case["window"]) for n, c in zip(new, ctx))))
    return {"bytes": 264.0 * keys * hkv + 512.0 * rows * hq + 4.0 * keys / PAGE + 8.0 * len(new),
            "flops": 4.0 * D * pairs * hq}


# --- from the definitions, in 64 bits

def _exact_pages(case, seed):
    s = _prepare_pages(case, _generator(seed))
    new, old, table = s["new"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    free, count, rows = s["free_pages"].tolist(), int(s["free_count"]), case["rows"]
    fits, wanted = [], 0
    for n, c in zip(new, old):                     # pages, in slot order
        need = _pages(c + n) - _pages(c) if c + n <= len(table[0]) * PAGE else -1
        wanted += max(need, 0)
        fits.append(n if need == 0 or (need > 0 and wanted <= count) else 0)
    cu, positions, slots, granted, asked, top = [0], [], [], [], 0, count
    for b, n in enumerate(fits):                   # rows, in slot order
        asked += n
        granted.append(n if asked <= rows else 0)
        for p in range(old[b], old[b] + granted[b]):
            if p % PAGE == 0:
                top -= 1
                table[b][p // PAGE] = free[top]
            positions.append(p)
            slots.append(table[b][p // PAGE] * PAGE + p % PAGE)
        cu.append(len(positions))
    pad = [-1] * (rows - len(positions))
    same = _prepare_pages(case, _generator(seed))  # the rollback undoes the step
    return [_int32(x) for x in (cu, positions + pad, slots + pad, granted)] + [
        same[name] for name in ("table", "lengths", "free_pages", "free_count")]


def _exact_append(case, seed):
    s = _prepare_append(case, _generator(seed))
    hq, hkv = case["q_heads"], case["kv_heads"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    p = s["positions"].long()
    c, sn = s["cos"].double()[p][:, None], s["sin"].double()[p][:, None]

    def turned(y, gain):
        y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain.double()
        a, b = y[..., :64], y[..., 64:]
        return torch.cat([a * c + b * sn, b * c - a * sn], -1)

    q, k, v = turned(x[:, :hq], s["q_gain"]), turned(x[:, hq:hq + hkv], s["k_gain"]), x[:, hq + hkv:]
    k = k.to(torch.bfloat16).double()               # the cache quantizes bf16 rows
    kv_scale = s["cache"]["kv_scale"].double()
    pages = [s["cache"][name].view(torch.float8_e4m3fn).double() for name in ("k_pages", "v_pages")]
    page, slot = s["slot_map"].long() // PAGE, s["slot_map"].long() % PAGE
    d = torch.arange(D, device=DEVICE)
    places = [(d % 32 // 16) * 1024 + (d // 32 * 16 + slot[:, None]) * 16 + d % 16,
              d // 64 * 1024 + (slot[:, None] // 4 * 16 + d % 16) * 16 + d // 16 % 4 * 4 + slot[:, None] % 4]
    for i, rows in enumerate((k, v)):
        scale = rows.abs().amax(-1) / FP8_MAX
        scale = torch.where(scale == 0, 1.0, scale)
        for h in range(hkv):
            codes = (rows[:, h] / scale[:, h, None]).to(torch.float8_e4m3fn).double()
            pages[i][page[:, None], h, places[i]] = codes
            kv_scale[page, h, i, slot] = scale[:, h]
    return [q, pages[0], pages[1], kv_scale]


def _exact_attend(case, seed):
    pairs = sum(n * (n + c) for n, c in zip(*_requests(case)))
    if pairs * case["q_heads"] > 3e9:
        return None
    s = _prepare_attend(case, _generator(seed))
    hq, hkv = case["q_heads"], case["kv_heads"]
    d, slot = torch.arange(D, device=DEVICE), torch.arange(PAGE, device=DEVICE)[:, None]
    at_k = (d % 32 // 16) * 1024 + (d // 32 * 16 + slot) * 16 + d % 16
    at_v = d // 64 * 1024 + (slot // 4 * 16 + d % 16) * 16 + d // 16 % 4 * 4 + slot % 4
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    row = 0
    for b, (n, length) in enumerate(zip(s["new"], s["lengths"])):
        pages = s["table"][b, :_pages(length)].long()
        scale = s["cache"]["kv_scale"][pages].double()
        keys = torch.arange(length, device=DEVICE)
        place = torch.arange(length - n, length, device=DEVICE)[:, None]
        hidden = (keys > place) | ((keys < place - case["window"]) if case["window"] >= 0 else False)
        for h in range(hkv):
            k = (s["cache"]["k_pages"][pages, h][:, at_k].view(torch.float8_e4m3fn).double() *
                 scale[:, h, 0, :, None]).flatten(0, 1)[:length]
            v = (s["cache"]["v_pages"][pages, h][:, at_v].view(torch.float8_e4m3fn).double() *
                 scale[:, h, 1, :, None]).flatten(0, 1)[:length]
            for head in range(h * hq // hkv, (h + 1) * hq // hkv):
                z = s["q"][row:row + n, head].double() @ k.t() / math.sqrt(D)
                out[row:row + n, head] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v
        row += n
    return out


def _exact_sample(case, seed):
    s = _prepare_sample(case, _generator(seed))
    tokens = []
    for r in range(case["rows"]):
        z = s["logits"][r].double()
        ids = torch.arange(z.numel(), device=DEVICE)
        if s["mask"] is not None:
            words = s["mask"][r].long() & 0xFFFFFFFF
            ids = ids[(words[ids // 32] >> (ids % 32)) & 1 == 1]
        z = z[ids]
        if not ids.numel():
            tokens.append(-1)
            continue
        temperature, k = float(s["temperature"][r]), int(s["top_k"][r])
        if temperature <= 0:
            tokens.append(int(ids[(z == z.max()).nonzero()[0, 0]]))
            continue
        if 0 < k < z.numel():
            least = z.topk(k).values[-1]
            equal = (z == least) & ((z == least).cumsum(0) <= k - (z > least).sum())
            ids, z = ids[(z > least) | equal], z[(z > least) | equal]
        w = torch.exp((z - z.max()) / temperature)
        levels, which = torch.unique(w, return_inverse=True)
        mass = torch.zeros_like(levels).index_add_(0, which, w)
        above = mass.flip(0).cumsum(0).flip(0) - mass
        p = float(s["top_p"][r])
        keep = ((above < p * w.sum()) | (levels == 1) if p < 1 else torch.ones_like(levels, dtype=torch.bool))[which]
        keep &= w >= float(s["min_p"][r])
        share = w[keep].cumsum(0)
        tokens.append(int(ids[keep][int((share <= float(s["uniform"][r]) * share[-1]).sum())]))
    return _int32(tokens)


def exact(case, seed):
    return {"pages": _exact_pages, "append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["kind"]](case, seed)
