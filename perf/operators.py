"""Measured cases of the long-sequence attention operators.

Three operators that are used together when a Transformer runs over whole scenes (the tokens of many agents packed into long
rows) instead of one short history per agent:

* ``rope``: RMS norm of queries and keys per head with the rotation of their positions in the same pass;
* ``attn``: attention with capped scores, a bias linear in the distance, document and prefix masks, cache lengths;
* ``rel``:  the same attention with a bias learned per head and distance bucket, and its gradient.

``run`` computes one pass of a case: in elementary torch operations where ``own`` is false, through the framework's entry points
(``multimodal_transformer_amd.torch_ops``) where it is true.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------------ cases
def _rope(name, dtype, B, L, H, Hk, dh, rot, interleaved, far, train):
    return {"name": name, "op": "rope", "dtype": dtype, "B": B, "L": L, "H": H, "Hk": Hk, "dh": dh, "rot": rot,
            "interleaved": interleaved, "far": far, "train": train}


def _attn(name, op, dtype, B, Lq, Lk, H, Hk, dh, causal, train, softcap=0.0, slopes=False, docs=0, prefix=False, cache=False,
          buckets=0, reach=0):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "dh": dh, "causal": causal,
            "train": train, "softcap": softcap, "slopes": slopes, "docs": docs, "prefix": prefix, "cache": cache,
            "buckets": buckets, "reach": reach}


def listed():
    return [
        # one new token for each of 32 requests at far positions: the call before every attention step of a decode loop
        _rope("rope_one_token", "bf16", 32, 1, 16, 4, 128, 128, False, 100000, False),
        # a training step of a bf16 model with 16 query and 4 key heads
        _rope("rope_train", "bf16", 4, 4096, 16, 4, 128, 128, False, 0, True),
        # the framework's own heads (8 of 32) in fp32, odd rows, half of each head turned, neighbouring pairs
        _rope("rope_fp32_ragged", "fp32", 3, 1037, 8, 8, 32, 16, True, 0, True),
        # a batch of agents: 9 observed and 12 future tokens, history visible to all, future causal, 8 heads of 32 in fp32
        _attn("attn_agents_fp32", "attn", "fp32", 128, 21, 21, 8, 8, 32, True, True, prefix=True),
        # one new token against a short cache: latency
        _attn("attn_one_token_short", "attn", "bf16", 4, 1, 517, 8, 8, 64, True, False, cache=True),
        # one new token for each of 16 requests against long ragged caches, capped scores: the cache is read once
        _attn("attn_one_token_long", "attn", "bf16", 16, 1, 32768, 32, 8, 128, True, False, softcap=30.0, cache=True),
        # a chunk of 64 new tokens against a long cache, bias linear in the distance
        _attn("attn_chunk", "attn", "fp16", 2, 64, 16384, 16, 4, 128, True, False, slopes=True, cache=True),
        # training on rows into which several scenes are packed
        _attn("attn_scenes_train", "attn", "bf16", 2, 4096, 4096, 16, 4, 64, True, True, slopes=True, docs=7),
        # training with a prefix that everybody sees, capped scores, an odd length
        _attn("attn_prefix_train", "attn", "bf16", 4, 2111, 2111, 16, 16, 128, True, True, softcap=50.0, prefix=True),
        # an encoder: bidirectional buckets
        _attn("rel_encoder_train", "rel", "bf16", 2, 2048, 2048, 16, 16, 64, False, True, buckets=32, reach=128),
        # odd length, odd head size, shared key heads, fp16
        _attn("rel_fp16_ragged", "rel", "fp16", 3, 1333, 1333, 8, 2, 80, True, True, buckets=32, reach=256),
        # the longest training row
        _attn("rel_long_train", "rel", "bf16", 1, 8192, 8192, 16, 4, 128, True, True, buckets=32, reach=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _unnamed(case):
    del case["name"]
    return case


def draw(rng):
    kind = rng.choice(["rope", "rope", "train", "train", "rel", "rel", "serve", "serve"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "rope":
        dh = rng.choice([32, 64, 80, 96, 128])
        Hk = rng.choice([1, 2, 4, 8])
        H = Hk * rng.choice([1, 2, 4])
        L = rng.choice([1, _log_int(rng, 2, 4096)])
        B = _log_int(rng, 1, max(1, min(64, 4 * 4096 * 16 // (L * H))))
        return _unnamed(_rope("", dtype, B, L, H, Hk, dh, rng.choice([dh, dh // 2]), rng.random() < 0.4,
                              rng.choice([0, 1000, 100000]), rng.random() < 0.6))
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if kind == "serve":
        Lk = _log_int(rng, 16, 32768)
        Lq = min(Lk, rng.choice([1, 1, 2, _log_int(rng, 2, 128)]))
        B = _log_int(rng, 1, max(1, min(64, 16 * 32768 * 8 // (Lk * Hk * (2 if dtype == "fp32" else 1)) // max(1, Lq // 16))))
        return _unnamed(_attn("", "attn", dtype, B, Lq, Lk, H, Hk, dh, True, False, softcap=softcap, slopes=rng.random() < 0.4,
                              cache=True))
    top = 2048 if dtype == "fp32" else 4096
    L = _log_int(rng, 17, top)
    most = max(1, int(2 * 4096 * 4096 * 8 / (L * L * H) / (8 if dtype == "fp32" else 1)))
    B = _log_int(rng, 1, min(64, most))
    causal = rng.random() < 0.6
    if kind == "train":
        return _unnamed(_attn("", "attn", dtype, B, L, L, H, Hk, dh, causal, True, softcap=softcap, slopes=rng.random() < 0.5,
                              docs=rng.choice([0, 0, 2, 5, 9]), prefix=causal and rng.random() < 0.5))
    return _unnamed(_attn("", "rel", dtype, B, L, L, H, Hk, dh, causal, True, softcap=softcap, docs=rng.choice([0, 0, 3]),
                          buckets=rng.choice([16, 32]), reach=rng.choice([64, 128, 256])))


# ------------------------------------------------------------------------------------- what follows from a case alone
def _document_lengths(L, n):
    """n documents and, at the end of the row, some padding (about 3 %)."""
    n = max(1, min(n, L // 4))
    weights = [0.35 + ((i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]
    room = L - L // 32
    total = sum(weights)
    lens = [max(1, int(room * w / total)) for w in weights]
    return lens, L - sum(lens)


def _cache_lengths(B, Lq, Lk):
    """Lengths between about a quarter of the cache and all of it; the first request fills it."""
    out = []
    for b in range(B):
        f = 1.0 if b == 0 else 0.25 + 0.75 * ((b * 0.6180339887498949) % 1.0)
        out.append(max(Lq, min(Lk, int(Lk * f))))
    return out


def _prefixes(B, L):
    return [int(L * (0.2 + 0.3 * ((b + 1) * 0.7548776662466927 % 1.0))) for b in range(B)]


def _pairs(case):
    """Visible (query, key) pairs of all batch rows, for one head."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]

    def tri(n_q, n_k):                       # the last n_q of n_k positions, each seeing itself and what is before it
        return n_q * (n_k - n_q) + n_q * (n_q + 1) // 2

    if case["cache"]:
        return sum(tri(Lq, n) if case["causal"] else Lq * n for n in _cache_lengths(B, Lq, Lk))
    spans = _document_lengths(Lk, case["docs"])[0] if case["docs"] else [Lk]
    prefixes = _prefixes(B, Lk) if case["prefix"] else [0] * B
    total = 0
    for p in prefixes:
        start = 0
        for n in spans:
            if not case["causal"]:
                total += n * n
            else:
                inside = max(0, min(n, p - start))                   # prefix positions of this document
                total += tri(n, n) + inside * (inside - 1) // 2
            start += n
    return total


def work(case):
    e = _BYTES[case["dtype"]]
    B, H, Hk, dh = case["B"], case["H"], case["Hk"], case["dh"]
    if case["op"] == "rope":
        n = B * case["L"] * (H + Hk) * dh
        extra = B * case["L"] * 8 + case["rot"] * 4 + 2 * dh * e
        if case["train"]:                    # x, y; x, gy, dx; weights and their gradients
            return {"bytes": 5 * n * e + 2 * extra + 2 * dh * e, "flops": 22 * n}
        return {"bytes": 2 * n * e + extra, "flops": 8 * n}
    pairs = _pairs(case)
    nq = B * case["Lq"] * H * dh
    nk = (sum(_cache_lengths(B, case["Lq"], case["Lk"])) if case["cache"] else B * case["Lk"]) * Hk * dh
    if case["train"]:                        # q k v o; q k v o do dq dk dv
        return {"bytes": (6 * nq + 6 * nk) * e, "flops": 14 * dh * pairs * H}
    return {"bytes": (2 * nq + 2 * nk) * e, "flops": 4 * dh * pairs * H}


def _bucket_table(buckets, reach, both):
    """Bucket of each distance j - i in -reach..reach: every near distance has its own, far ones share them by their logarithm.
    In whole numbers, so that no distance falls on the wrong side of a border."""
    half = buckets // 2 if both else buckets
    near = half // 2
    bins = half - near

    def one(d):
        if d < near:
            return d
        m = 0
        while m + 1 < bins and d ** bins * near ** (m + 1) >= reach ** (m + 1) * near ** bins:
            m += 1
        return near + m

    out = []
    for r in range(-reach, reach + 1):
        if r > 0:
            out.append(half + one(r) if both else 0)
        else:
            out.append(one(-r))
    return out


# ------------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(case, seed):
    """The tensors of a case, on the GPU."""
    g = _generator(seed)
    dt = _TYPES[case["dtype"]]
    dev = torch.device("cuda")
    B, H, Hk, dh = case["B"], case["H"], case["Hk"], case["dh"]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    t = {}
    if case["op"] == "rope":
        L, rot = case["L"], case["rot"]
        qkv = normal(B, L, H + 2 * Hk, dh)                # one projection's output; queries and keys are views of it
        t["q"], t["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        t["q_weight"] = (1.0 + 0.2 * torch.randn(dh, generator=g, device=dev)).to(dt)
        t["k_weight"] = (1.0 + 0.2 * torch.randn(dh, generator=g, device=dev)).to(dt)
        t["inv_freq"] = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        first = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device=dev)
        t["positions"] = first + torch.arange(L, device=dev)
        if case["train"]:
            t["gq"], t["gk"] = normal(B, L, H, dh), normal(B, L, Hk, dh)
        return t
    Lq, Lk = case["Lq"], case["Lk"]
    t["q"] = normal(B, Lq, H, dh)
    t["k"] = normal(B, Lk, Hk, dh)
    t["v"] = normal(B, Lk, Hk, dh)
    if case["cache"]:
        t["kv_len"] = torch.tensor(_cache_lengths(B, Lq, Lk), dtype=torch.int32, device=dev)
    if case["docs"]:
        lens, pad = _document_lengths(Lk, case["docs"])
        ids = [i for i, n in enumerate(lens) for _ in range(n)] + [-1] * pad
        t["doc"] = torch.tensor(ids, dtype=torch.int32, device=dev).expand(B, Lk).contiguous()
    if case["prefix"]:
        t["prefix"] = torch.tensor(_prefixes(B, Lk), dtype=torch.int32, device=dev)
    if case["slopes"]:
        t["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=dev)
    if case["buckets"]:
        t["rel_buckets"] = torch.tensor(_bucket_table(case["buckets"], case["reach"], not case["causal"]), dtype=torch.int32,
                                        device=dev)
        t["rel_bias"] = torch.randn(H, case["buckets"], generator=g, device=dev) * 0.5
    if case["train"]:
        t["go"] = normal(B, Lq, H, dh)
    return t


def prepare(case, seed):
    t = _values(case, seed)
    if case["train"]:
        for name in ("q", "k", "v", "q_weight", "k_weight", "rel_bias"):
            if name in t:
                t[name] = t[name].detach().requires_grad_()
    return case, t


# ------------------------------------------------------------------------------------------------------------------ plain
def _plain_turn(x, weight, cos, sin, eps, interleaved):
    x = x.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    half = cos.shape[-1]
    if interleaved:
        a, b = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
    else:
        a, b = n[..., :half], n[..., half:2 * half]
    ya, yb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    return torch.cat((turned, n[..., 2 * half:]), -1)


def _plain_rope(case, t):
    angle = t["positions"].double()[..., None] * t["inv_freq"]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    dt = t["q"].dtype
    return (_plain_turn(t["q"], t["q_weight"], cos, sin, 1e-6, case["interleaved"]).to(dt),
            _plain_turn(t["k"], t["k_weight"], cos, sin, 1e-6, case["interleaved"]).to(dt))


class _BiasOfBuckets(torch.autograd.Function):
    """table (H, n) at bucket (Lq, Lk) -> (H, Lq, Lk), bucket a function of j - i.  The gradient of an entry is a sum over up to
    millions of pairs: in 64 bits, first along the diagonals (laid out as columns by one more element per row), then by bucket."""

    @staticmethod
    def forward(ctx, table, bucket):
        ctx.save_for_backward(bucket)
        ctx.entries = table.shape[1]
        return table[:, bucket]

    @staticmethod
    def backward(ctx, grad):
        bucket, = ctx.saved_tensors
        H, Lq, Lk = grad.shape
        W = Lq + Lk
        skewed = torch.nn.functional.pad(grad, (0, Lq)).view(H, Lq * W)
        skewed = torch.nn.functional.pad(skewed, (0, Lq)).view(H, Lq, W + 1)
        diagonals = skewed.sum(1, dtype=torch.float64)                       # (j - i) mod (W + 1)
        where = torch.cat((bucket[0], bucket[:, 0].flip(0)))                 # bucket of j - i = 0 .. Lk - 1, then of -(Lq - 1) .. 0
        sums = torch.zeros(H, ctx.entries, dtype=torch.float64, device=grad.device)
        values = torch.cat((diagonals[:, :Lk], diagonals[:, W + 2 - Lq:], torch.zeros_like(sums[:, :1])), 1)
        return sums.index_add_(1, where, values).float(), None


def _plain_attention(case, t):
    B, Lq, H, dh = t["q"].shape
    Lk, Hk = t["k"].shape[1:3]
    G = H // Hk
    dev = t["q"].device
    q = t["q"].float().view(B, Lq, Hk, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, dh)
    k = t["k"].float().permute(0, 2, 3, 1).contiguous()
    v = t["v"].float().permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q, k).view(B, Hk, G, Lq, Lk) * (1.0 / math.sqrt(dh))
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    length = t["kv_len"].long() if "kv_len" in t else torch.full((B,), Lk, device=dev)
    at = (length - Lq)[:, None] + torch.arange(Lq, device=dev)
    there = torch.arange(Lk, device=dev)
    apart = there - at[:, :, None]                                                        # (B, Lq, Lk)
    if "slopes" in t:
        s = s - t["slopes"].view(1, Hk, G, 1, 1) * apart.abs().float()[:, None, None]
    if "rel_bias" in t:
        reach = case["reach"]
        bucket = t["rel_buckets"].long()[apart[0].clamp(-reach, reach) + reach]            # the same for every row: no cache here
        s = s + _BiasOfBuckets.apply(t["rel_bias"], bucket).view(1, Hk, G, Lq, Lk)
    seen = (there < length[:, None])[:, None, :].expand(B, Lq, Lk)
    if case["causal"]:
        before = apart <= 0
        if "prefix" in t:
            before = before | (there < t["prefix"].long()[:, None])[:, None]
        seen = seen & before
    if "doc" in t:
        seen = seen & (t["doc"][:, :, None] == t["doc"][:, None, :]) & (t["doc"] >= 0)[:, :, None]
    seen = seen[:, None, None]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0.0, 1.0)
    o = torch.matmul(p.view(B, Hk, G * Lq, Lk), v).view(B, Hk, G, Lq, dh)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Lq, H, dh).to(t["q"].dtype)


# ------------------------------------------------------------------------------------------------------------------ run
def _forward(case, t):
    if not own:
        return _plain_rope(case, t) if case["op"] == "rope" else _plain_attention(case, t)
    from multimodal_transformer_amd import torch_ops
    if case["op"] == "rope":
        return torch_ops.qk_norm_rope(t["q"], t["k"], t["q_weight"], t["k_weight"], t["inv_freq"], t["positions"], eps=1e-6,
                                      interleaved=case["interleaved"])
    return torch_ops.long_attention(t["q"], t["k"], t["v"], causal=case["causal"], prefix=t.get("prefix"), q_doc=t.get("doc"),
                                    k_doc=t.get("doc"), kv_len=t.get("kv_len"), softcap=case["softcap"], slopes=t.get("slopes"),
                                    rel_bias=t.get("rel_bias"), rel_buckets=t.get("rel_buckets"))


def run(state):
    case, t = state
    if not case["train"]:
        with torch.no_grad():
            return _forward(case, t)
    out = _forward(case, t)
    if case["op"] == "rope":
        grads = torch.autograd.grad(out, (t["q"], t["k"], t["q_weight"], t["k_weight"]), (t["gq"], t["gk"]))
        return tuple(x.detach() for x in out) + grads
    leaves = [t["q"], t["k"], t["v"]] + ([t["rel_bias"]] if "rel_bias" in t else [])
    return (out.detach(),) + torch.autograd.grad(out, leaves, t["go"])


# ------------------------------------------------------------------------------------------------------------------ exact
def _exact_head(x, w, gy, ang, interleaved):
    """One tensor of the rope case: the turned norm and, with gy, the gradients of x and w."""
    x, w = x.double(), w.double()
    dh, half = x.shape[-1], ang.shape[-1]
    idx = torch.arange(half, device=x.device)
    ia, ib = (2 * idx, 2 * idx + 1) if interleaved else (idx, idx + half)
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    r = (x.pow(2).sum(-1, keepdim=True) / dh + 1e-6).pow(-0.5)
    hat = x * r
    y = hat * w
    na, nb = y[..., ia], y[..., ib]
    y[..., ia], y[..., ib] = na * c - nb * s, na * s + nb * c
    if gy is None:
        return y, None, None
    g = gy.double()
    ga, gb = g[..., ia], g[..., ib]
    g[..., ia], g[..., ib] = ga * c + gb * s, gb * c - ga * s
    dw = (g * hat).sum((0, 1, 2))
    g = g * w
    return y, r * (g - hat * (g * hat).sum(-1, keepdim=True) / dh), dw


def _exact_attention(case, t):
    q, k, v = t["q"], t["k"], t["v"]
    B, Lq, H, dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    dev, cap, scale = q.device, case["softcap"], dh ** -0.5
    train = case["train"]
    o = torch.zeros(B, Lq, H, dh, dtype=torch.float64, device=dev)
    dq, dk, dv = torch.zeros_like(o), torch.zeros(k.shape, dtype=torch.float64, device=dev), \
        torch.zeros(k.shape, dtype=torch.float64, device=dev)
    dtable = torch.zeros(H, max(1, case["buckets"]), dtype=torch.float64, device=dev)
    j = torch.arange(Lk, device=dev)
    for b in range(B):
        n = int(t["kv_len"][b]) if "kv_len" in t else Lk
        i = torch.arange(Lq, device=dev)[:, None] + (n - Lq)
        hidden = (j >= n)[None].expand(Lq, Lk)
        if case["causal"]:
            later = j[None] > i
            if "prefix" in t:
                later = later & (j >= int(t["prefix"][b]))[None]
            hidden = hidden | later
        if "doc" in t:
            d = t["doc"][b]
            hidden = hidden | (d[:, None] != d[None]) | (d < 0)[:, None]
        empty = hidden.all(-1)
        far = i - j
        which = t["rel_buckets"].long()[(-far).clamp(-case["reach"], case["reach"]) + case["reach"]] if case["buckets"] else None
        for h in range(H):
            kh, vh = k[b, :, h // (H // Hk)].double(), v[b, :, h // (H // Hk)].double()
            kh, vh = torch.where((j < n)[:, None], kh, 0.0), torch.where((j < n)[:, None], vh, 0.0)
            qh = q[b, :, h].double()
            u = scale * (qh @ kh.t().contiguous())
            if cap:
                th = (u / cap).tanh()
                u = cap * th
            if case["slopes"]:
                u = u - far.abs() * float(t["slopes"][h].double())
            if which is not None:
                u = u + t["rel_bias"][h].double()[which]
            p = torch.softmax(u.masked_fill(hidden, -math.inf), -1).masked_fill(empty[:, None], 0.0)
            o[b, :, h] = p @ vh
            if not train:
                continue
            g = t["go"][b, :, h].double()
            du = g @ vh.t().contiguous()
            dv[b, :, h // (H // Hk)] += p.t().contiguous() @ g
            du = p * (du - (p * du).sum(-1, keepdim=True))
            if which is not None:
                dtable[h] += torch.bincount(which.flatten(), weights=du.flatten(), minlength=case["buckets"])
            if cap:
                du = du * (1.0 - th * th)
            dq[b, :, h] = scale * (du @ kh)
            dk[b, :, h // (H // Hk)] += scale * (du.t().contiguous() @ qh)
    if not train:
        return o
    return (o, dq, dk, dv) + ((dtable,) if case["buckets"] else ())


def exact(case, seed):
    t = _values(case, seed)
    with torch.no_grad():
        if case["op"] == "rope":
            ang = t["positions"].double()[..., None] * t["inv_freq"]
            q = _exact_head(t["q"], t["q_weight"], t.get("gq"), ang, case["interleaved"])
            k = _exact_head(t["k"], t["k_weight"], t.get("gk"), ang, case["interleaved"])
            return (q[0], k[0]) if not case["train"] else (q[0], k[0], q[1], k[1], q[2], k[2])
        if _pairs(case) * case["H"] * case["dh"] > 1 << 40:
            return None
        return _exact_attention(case, t)
