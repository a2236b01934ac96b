"""The attention operators' cases: what a serving program calls after the
selection, in their plain form (elementary torch operations in 32 bits) and
through the framework's kernels.

  slots   latent attention (absorbed form) of each query row over its own list of
          selected cache slots
  pages   latent attention (absorbed form) of each row over its whole paged cache
  prompt  latent attention (expanded form): ragged prompts, causal
  store   new tokens' keys and values into the paged 8-bit cache
  attend  grouped-query attention of each row over the paged 8-bit cache
"""
import importlib
import math

import torch

own = False

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one request's decode row over a small selection (the default index budget of 512): latency
        dict(name="slots one row", op="slots", rows=1, heads=64, top=512, slots=65536, dtype="bf16"),
        # the decode batch: 128 requests, Top-2048 each, cache far above the L2
        dict(name="slots decode batch", op="slots", rows=128, heads=64, top=2048, slots=2097152, dtype="bf16"),
        # a prompt chunk of one long request, every row with a selection of its own; two groups of heads
        dict(name="slots prompt chunk", op="slots", rows=1024, heads=128, top=2048, slots=123904, dtype="bf16"),
        # one long context before any selection: the work of a single row spread over the GPU
        dict(name="pages one long row", op="pages", rows=1, heads=64, longest=131072, shortest=131072, dtype="bf16"),
        # a ragged decode batch over the whole cache, half-precision, a head count that fills no tile
        dict(name="pages ragged batch", op="pages", rows=48, heads=24, longest=16384, shortest=1, dtype="fp16"),
        # a short prompt: latency
        dict(name="prompt short", op="prompt", heads=16, requests=1, queries=203, prefix=0, dtype="bf16"),
        # several ragged prompts after a cached prefix each
        dict(name="prompt ragged prefix", op="prompt", heads=32, requests=5, queries=1531, prefix=4096, dtype="fp16"),
        # one long prompt: the tensor cores' case
        dict(name="prompt long", op="prompt", heads=32, requests=1, queries=8192, prefix=0, dtype="bf16"),
        # one decode step of 128 requests: a token each into part-filled pages
        dict(name="store decode step", op="store", requests=128, tokens=128, prefix=4096, heads=8, dtype="bf16"),
        # prompts of several requests, into pages that earlier tokens may have begun
        dict(name="store prompts", op="store", requests=4, tokens=16384, prefix=1024, heads=8, dtype="bf16"),
        # one short decode row: latency
        dict(name="attend one row", op="attend", rows=1, heads=32, kv_heads=4, longest=4097, shortest=4097, dtype="bf16"),
        # a ragged decode batch over caches of up to 16K tokens
        dict(name="attend decode batch", op="attend", rows=64, heads=32, kv_heads=4, longest=16384, shortest=1024, dtype="bf16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["slots", "pages", "prompt", "store", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "slots":
        top, heads = spread(1, 2048), spread(1, 128)
        rows = spread(1, max(1, min(1024, (1 << 27) // (top * heads))))
        return dict(op=op, rows=rows, heads=heads, top=top, slots=spread(4096, 300000), dtype=dtype)
    if op == "pages":
        rows, heads = spread(1, 128), spread(1, 128)
        longest = spread(1, min(131072, (1 << 20) // rows))
        return dict(op=op, rows=rows, heads=heads, longest=longest, shortest=spread(1, longest), dtype=dtype)
    if op == "prompt":
        queries, heads = spread(1, 6000), spread(1, 64)
        prefix = rng.choice([0, spread(1, 4096)])
        requests = spread(1, min(queries, 24))
        while heads > 1 and heads * queries * (queries + prefix * requests) > (1 << 30):
            heads //= 2
        while prefix and heads * queries * (queries + prefix * requests) > (1 << 30):
            prefix //= 2
        return dict(op=op, heads=heads, requests=requests, queries=queries, prefix=prefix, dtype=dtype)
    if op == "store":
        requests = spread(1, 200)
        return dict(op=op, requests=requests, tokens=spread(requests, 16384), prefix=spread(1, min(8192, 200000 // requests)),
                    heads=rng.choice([1, 2, 3, 4, 8]), dtype=dtype)
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    rows = spread(1, 128)
    longest = spread(1, min(131072, (1 << 22) // (rows * kv_heads)))
    return dict(op=op, rows=rows, heads=kv_heads * spread(1, 20), kv_heads=kv_heads, longest=longest,
                shortest=spread(1, longest), dtype=dtype)


# -- inputs ------------------------------------------------------------------
def _counts(total, parts):
    """`total` split into `parts` uneven counts of at least one."""
    w = [1 + (7 * i) % 5 for i in range(parts)]
    got = [1 + (total - parts) * x // sum(w) for x in w]
    got[0] += total - sum(got)
    return got


def _ends(counts):
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    return ends


def _lens(case):
    """The rows' lengths: spread evenly from the shortest to the longest, in a mixed order."""
    n, lo, hi = case["rows"], case["shortest"], case["longest"]
    return [lo + (hi - lo) * ((i * 7919) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _prompt_plan(case):
    q = _counts(case["queries"], case["requests"])
    k = [n + case["prefix"] - (case["prefix"] * i) // (2 * len(q)) for i, n in enumerate(q)]
    return _ends(q), _ends(k)


def _store_plan(case):
    counts = _counts(case["tokens"], case["requests"])
    prefix = [case["prefix"] - (case["prefix"] * ((i * 31) % 17)) // 17 for i in range(case["requests"])]
    return counts, prefix


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, dt = case["op"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dt)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def pages(count):
        return torch.randperm(count, generator=g, device=dev).to(torch.int32)

    s = {"case": dict(case)}
    if op in ("slots", "pages"):
        s["q"] = normal(case["rows"], case["heads"], 576)
        s["scale"] = 192 ** -0.5
    if op == "slots":
        s["pool"] = normal(case["slots"], 1, 576)
        ids = torch.randint(0, case["slots"], (case["rows"], case["top"]), generator=g, device=dev, dtype=torch.int32)
        ids = ids.sort(dim=1).values
        if case["rows"] > 2:
            ids[1, case["top"] // 3:] = -1      # a row that is still short
        s["ids"] = ids
    elif op == "pages":
        lens = _lens(case)
        width = -(-case["longest"] // PAGE)
        s["pool"] = normal(case["rows"] * width * PAGE, 1, 576)
        s["table"] = pages(case["rows"] * width).view(case["rows"], width)
        s["lens"] = ints(lens)
    elif op == "prompt":
        qe, ke = _prompt_plan(case)
        h = case["heads"]
        s["q"] = normal(qe[-1], h, 192)
        kv = normal(ke[-1], h, 256)              # one projection's output: keys and values side by side
        s["k"], s["v"] = kv[..., :128], kv[..., 128:]
        s["k_rope"] = normal(ke[-1], 576)[:, 512:]   # the last columns of the latent rows
        s["offsets"], s["kv_offsets"] = ints(qe), ints(ke)
        s["scale"] = 192 ** -0.5
    else:
        h = case["heads"] if op == "store" else case["kv_heads"]
        if op == "store":
            counts, prefix = _store_plan(case)
            ends = [p + c for p, c in zip(prefix, counts)]
            width = -(-max(ends) // PAGE)
            rows = case["requests"]
            s["k"], s["v"] = normal(case["tokens"], h, 128), normal(case["tokens"], h, 128) * 0.5
            s["prefix"], s["offsets"] = ints(prefix), ints(_ends(counts))
            s["span"] = max((e - 1) // PAGE - p // PAGE + 1 for e, p in zip(ends, prefix))
        else:
            width = -(-case["longest"] // PAGE)
            rows = case["rows"]
            s["q"] = normal(rows, case["heads"], 128)
            s["lens"] = ints(_lens(case))
            s["scale"] = 128 ** -0.5
        n = rows * width
        s["table"] = pages(n).view(rows, width)
        # keys and values as an earlier store left them: codes up to 448 under power-of-two scales
        for x, spread in (("k", 3), ("v", 4)):
            s[x + "_scale"] = torch.exp2(torch.randint(-8, spread - 8, (n, h), generator=g, device=dev).float())
            codes = torch.empty((n, h, PAGE, 128), device=dev, dtype=E4M3)
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                codes[a:b] = (torch.randn((b - a, h, PAGE, 128), generator=g, device=dev) * 90).clamp(-448, 448).to(E4M3)
            s[x + "_cache"] = codes
    return s


# -- one pass ----------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"slots": _slots, "pages": _pages, "prompt": _prompt, "store": _store, "attend": _attend}[op](state)


def _own(op, s):
    if op == "slots":
        latent = importlib.import_module("10_20_b200.latent_attention")
        return latent.attend_slots(s["q"], s["pool"], None, s["ids"], s["scale"])
    if op == "pages":
        latent = importlib.import_module("10_20_b200.latent_attention")
        return latent.attend_pages(s["q"], s["pool"], s["table"], s["lens"], s["scale"])
    if op == "prompt":
        latent = importlib.import_module("10_20_b200.latent_attention")
        return latent.attend_prompt(s["q"], s["k"], s["k_rope"], s["v"], s["offsets"], s["scale"],
                                    kv_offsets=s["kv_offsets"])
    kv8 = importlib.import_module("10_20_b200.kv8")
    cache = (s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"])
    if op == "store":
        kv8.store(*cache, s["k"], s["v"], s["table"], s["prefix"], s["offsets"])
        return cache
    return kv8.attend(s["q"], *cache, s["table"], s["lens"], s["scale"])


def _weights(scores, live):
    """exp(scores - row maximum) with masked places zero, its sums, and the logarithm of the sums of exp(scores)."""
    scores = scores.masked_fill_(~live, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    return e, total, (total.log() + top).squeeze(-1)


def _latent(q, kv, live, scale):
    """rows x heads over rows x tokens of 576, the first 512 of which are the values too."""
    e, total, lse = _weights(torch.matmul(q.float(), kv.transpose(1, 2)).mul_(scale), live[:, None])
    out = torch.matmul(e, kv[..., :512]) / torch.where(total > 0, total, 1.0)
    return out.to(q.dtype), lse


def _slots(s):
    ids = s["ids"]
    kv = s["pool"][ids.clamp(min=0).long(), 0].float()
    return _latent(s["q"], kv, ids >= 0, s["scale"])


def _pages(s):
    rows, width = s["table"].shape
    kv = s["pool"].view(-1, PAGE, 576)[s["table"].long()].view(rows, width * PAGE, 576).float()
    live = torch.arange(width * PAGE, device=kv.device) < s["lens"][:, None]
    return _latent(s["q"], kv, live, s["scale"])


def _prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    dev = q.device
    qe, ke = s["offsets"].long(), s["kv_offsets"].long()
    i, j = torch.arange(q.shape[0], device=dev), torch.arange(k.shape[0], device=dev)
    qr, kr = (i[:, None] >= qe[1:]).sum(1), (j[:, None] >= ke[1:]).sum(1)
    last = (i - qe[qr]) + (ke[qr + 1] - ke[qr]) - (qe[qr + 1] - qe[qr])      # the last key that the query sees
    live = (qr[:, None] == kr) & ((j - ke[kr]) <= last[:, None])
    rope = s["k_rope"].float()[:, None].expand(-1, k.shape[1], -1)
    keys = torch.cat([k, rope], -1).permute(1, 2, 0)
    e, total, lse = _weights(torch.matmul(q.transpose(0, 1), keys).mul_(s["scale"]), live)
    out = torch.matmul(e, v.transpose(0, 1)) / torch.where(total > 0, total, 1.0)
    return out.transpose(0, 1).to(s["q"].dtype).contiguous(), lse.t().contiguous()


def _scale_of(most):
    """The smallest power of two 2^e, -40 <= e <= 40, with 448 * 2^e >= most."""
    m, x = torch.frexp(most)
    e = torch.where(m <= 0.875, x - 9, x - 8).clamp(-40, 40)
    return torch.exp2(torch.where(most > 0, e, -40).float())


def _store(s):
    offsets, prefix = s["offsets"].long(), s["prefix"].long()
    counts = offsets[1:] - offsets[:-1]
    table, dev = s["table"].long(), prefix.device
    index = prefix[:, None] // PAGE + torch.arange(s["span"], device=dev)
    at = index[..., None] * PAGE + torch.arange(PAGE, device=dev)            # requests x pages x 64 positions
    fresh = (at >= prefix[:, None, None]) & (at < (prefix + counts)[:, None, None])
    earlier = at < prefix[:, None, None]
    touched = fresh.any(-1)
    rows = (offsets[:-1, None, None] + at - prefix[:, None, None]).clamp(0, s["k"].shape[0] - 1)
    page = table.gather(1, index.clamp(max=table.shape[1] - 1))
    for x in ("k", "v"):
        cache, scale = s[x + "_cache"], s[x + "_scale"]
        new = s[x][rows].float().transpose(2, 3)                             # requests x pages x heads x 64 x 128
        new_at = fresh[:, :, None, :, None]
        most = torch.where(new_at, new.abs(), 0.0).amax((-1, -2))
        old = scale[page]
        now = _scale_of(most)
        now = torch.where(earlier.any(-1)[..., None], torch.maximum(now, old), now)
        kept = cache[page]
        again = (kept.float() * (old / now)[..., None, None]).clamp(-448, 448).to(E4M3)
        code = (new / now[..., None, None]).clamp(-448, 448).to(E4M3)
        code = torch.where(new_at, code.view(torch.uint8), torch.where(earlier[:, :, None, :, None],
                           again.view(torch.uint8), kept.view(torch.uint8))).view(E4M3)
        cache.view(torch.uint8)[page[touched]] = code.view(torch.uint8)[touched]
        scale[page[touched]] = now[touched]
    return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _attend(s):
    q = s["q"].float()
    rows, heads, d = q.shape
    table = s["table"].long()
    kv_heads, width = s["k_cache"].shape[1], table.shape[1]

    def values(x):   # rows x kv_heads x tokens x 128
        t = s[x + "_cache"][table].float() * s[x + "_scale"][table][..., None, None]
        return t.transpose(1, 2).reshape(rows, kv_heads, width * PAGE, d)

    live = torch.arange(width * PAGE, device=q.device) < s["lens"][:, None]
    k = values("k")
    scores = torch.matmul(q.view(rows, kv_heads, heads // kv_heads, d), k.transpose(2, 3)).mul_(s["scale"])
    del k
    e, total, lse = _weights(scores, live[:, None, None])
    out = torch.matmul(e, values("v")) / torch.where(total > 0, total, 1.0)
    return out.view(rows, heads, d).to(s["q"].dtype), lse.reshape(rows, heads)


# -- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    if op == "slots":
        r, h, t = case["rows"], case["heads"], case["top"]
        n = r * t - (t - t // 3 if r > 2 else 0)
        seen = min(n, case["slots"])           # a slot that several rows name is read once
        return {"bytes": seen * 1152 + 4 * r * t + r * h * (1152 + 1024 + 4), "flops": 2 * h * n * (576 + 512)}
    if op == "pages":
        r, h, n = case["rows"], case["heads"], sum(_lens(case))
        return {"bytes": n * 1152 + n // 16 + r * h * (1152 + 1024 + 4), "flops": 2 * h * n * (576 + 512)}
    if op == "prompt":
        qe, ke = _prompt_plan(case)
        h = case["heads"]
        pairs = 0
        for i in range(case["requests"]):
            nq, nk = qe[i + 1] - qe[i], ke[i + 1] - ke[i]
            pairs += nq * (nk - nq) + nq * (nq + 1) // 2
        return {"bytes": qe[-1] * h * (384 + 256 + 4) + ke[-1] * (h * 512 + 128), "flops": 2 * h * pairs * (192 + 128)}
    if op == "store":
        counts, prefix = _store_plan(case)
        h, pages, begun = case["heads"], 0, 0
        for c, p in zip(counts, prefix):
            pages += (p + c - 1) // PAGE - p // PAGE + 1
            begun += 1 if p % PAGE else 0
        # the scales of the begun pages are read; their earlier codes only where the scale rises
        return {"bytes": 2 * h * (case["tokens"] * 128 * 3 + 4 * pages + 4 * begun), "flops": 4 * h * case["tokens"] * 128}
    r, h, kv, n = case["rows"], case["heads"], case["kv_heads"], sum(_lens(case))
    return {"bytes": n * kv * 256 + n * kv // 8 + r * h * (256 + 256 + 4), "flops": 4 * h * n * 128}


# -- the definition in 64 bits ---------------------------------------------------
def _row(q, keys, values, scale, live=None):
    """softmax attention of queries [heads, d] over keys [(heads,) n, d], in 64 bits."""
    s = (q.double() @ keys.double().transpose(-1, -2)) * scale
    if live is not None:
        s = s.masked_fill(~live, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.nan_to_num(torch.exp(s - lse[..., None]), nan=0.0)
    return p @ values.double(), lse


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("slots", "pages"):
        outs, lses = [], []
        for r in range(case["rows"]):
            if op == "slots":
                ids = s["ids"][r]
                rows = s["pool"][ids[ids >= 0].long(), 0]
            else:
                n = int(s["lens"][r])
                t = torch.arange(n, device="cuda")
                rows = s["pool"][s["table"][r].long()[t // PAGE] * PAGE + t % PAGE, 0]
            out, lse = _row(s["q"][r], rows, rows[:, :512], s["scale"])
            outs.append(out)
            lses.append(lse)
        return torch.stack(outs), torch.stack(lses)
    if op == "prompt":
        qe, ke = _prompt_plan(case)
        out = torch.zeros((qe[-1], case["heads"], 128), dtype=torch.float64, device="cuda")
        lse = torch.zeros((qe[-1], case["heads"]), dtype=torch.float64, device="cuda")
        for i in range(case["requests"]):
            nq, nk = qe[i + 1] - qe[i], ke[i + 1] - ke[i]
            live = torch.ones((nq, nk), dtype=torch.bool, device="cuda").tril(nk - nq)
            for h in range(case["heads"]):
                keys = torch.cat([s["k"][ke[i]:ke[i + 1], h], s["k_rope"][ke[i]:ke[i + 1]]], 1)
                o, x = _row(s["q"][qe[i]:qe[i + 1], h], keys, s["v"][ke[i]:ke[i + 1], h], s["scale"], live)
                out[qe[i]:qe[i + 1], h], lse[qe[i]:qe[i + 1], h] = o, x
        return out, lse
    if op == "store":
        return _exact_store(s, *_store_plan(case))
    outs, lses = [], []
    kv = case["kv_heads"]
    for r in range(case["rows"]):
        n = int(s["lens"][r])
        pages = s["table"][r, :-(-n // PAGE)].long()

        def tokens(x):
            t = s[x + "_cache"][pages].double() * s[x + "_scale"][pages].double()[..., None, None]
            return t.permute(1, 0, 2, 3).reshape(kv, -1, 128)[:, :n]

        out, lse = _row(s["q"][r].view(kv, -1, 128), tokens("k"), tokens("v"), s["scale"])
        outs.append(out.reshape(-1, 128))
        lses.append(lse.reshape(-1))
    return torch.stack(outs), torch.stack(lses)


def _exact_store(s, counts, prefix):
    """Page by page: the scales from the definition; the codes as a round trip of the values in 64 bits."""
    caches = []
    for x in ("k", "v"):
        cache, scale, begin = s[x + "_cache"].to(torch.float32), s[x + "_scale"].double(), 0
        for r, (n, p) in enumerate(zip(counts, prefix)):
            new = s[x][begin:begin + n].double()
            begin += n
            for page in range(p // PAGE, (p + n - 1) // PAGE + 1):
                lo, hi = max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
                part = new[lo - p:hi - p].transpose(0, 1)
                slot = int(s["table"][r, page])
                need = part.abs().amax((1, 2)) / 448
                now = torch.exp2(torch.ceil(torch.log2(need)).clamp(-40, 40))
                if lo > page * PAGE:
                    now = torch.maximum(now, scale[slot])
                    old = cache[slot, :, :lo - page * PAGE].double() * (scale[slot] / now)[:, None, None]
                    cache[slot, :, :lo - page * PAGE] = old.float().to(E4M3).float()
                scale[slot] = now
                code = (part / now[:, None, None]).float()
                cache[slot, :, lo - page * PAGE:hi - page * PAGE] = code.clamp(-448, 448).to(E4M3).float()
        caches += [cache, scale]
    return tuple(caches)
