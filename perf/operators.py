"""The operators of a serving loop over a cache held in 4 bits, as cases that can be timed: in plain torch, or through this
package's entry points.

* ``prompt``  attention over packed prompts of different lengths, causal, grouped heads, optionally behind a cached prefix;
* ``write``   tokens into the cache (4-bit codes, a scale and a minimum per 32 values) and back as the values they stand for;
* ``decode``  one query token per sequence over the cache, optionally adding up the probability that every key received;
* ``evict``   the last tokens and those with the largest added-up probability into a smaller cache.

A group of up to 32 neighbouring values of one token's row is stored as m = its minimum, s = (its maximum - m) / 15 rounded
down to the cache's 16-bit type, and codes c = round((x - m) / s), at most 15; it stands for c * s + m.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
GROUP = 32         # values that share a scale and a minimum
PAGE = 64          # rows of a page of the paged caches


def _case(name, kind, dtype, B, N, N_kv, D, S, **more):
    c = {"kind": kind, "dtype": dtype, "B": B, "N": N, "N_kv": N_kv, "D": D, "S": S, "prefix": 0, "new": 0,
         "weights": False, "paged": False, "keep": 0, "recent": 0}
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a few chat turns that arrive together: nothing but launch, call and one wave of short tiles
        _case("prompt-short", "prompt", "bfloat16", 4, 32, 8, 128, 200),
        # chunks of prompts whose beginnings are in the cache already: ragged, one head of K/V per query head, narrow heads
        _case("prompt-chunks", "prompt", "float16", 24, 16, 16, 64, 1500, prefix=777),
        # documents to be summarised, a full batch of long prompts
        _case("prompt-long", "prompt", "float16", 8, 32, 8, 128, 4096),
        # the write of a decoding step: one token per sequence into a paged cache
        _case("write-token", "write", "bfloat16", 8, 0, 8, 128, 2048, new=1, paged=True),
        # prompts of a model with heads of an odd width
        _case("write-ragged", "write", "float16", 5, 0, 12, 80, 1301, new=901),
        # a full batch of long prompts into empty caches
        _case("write-prompts", "write", "float16", 16, 0, 8, 128, 4096, new=4096),
        # a decoding step of a few interactive users: paged cache, short contexts, probabilities added up
        _case("decode-few", "decode", "bfloat16", 4, 32, 8, 128, 2048, weights=True, paged=True),
        # one head of K/V per query head, odd width, odd lengths
        _case("decode-odd", "decode", "float16", 7, 12, 12, 80, 3001),
        # a decoding step of a full serving batch with long contexts of different lengths
        _case("decode-full", "decode", "float16", 32, 32, 8, 128, 16384, weights=True),
        # a few users' caches are full: down to half
        _case("evict-few", "evict", "bfloat16", 4, 0, 8, 128, 2048, keep=1024, recent=128, paged=True),
        # odd sizes all over
        _case("evict-odd", "evict", "float16", 7, 0, 12, 80, 1501, keep=703, recent=33),
        # a full serving batch after its prompts: half of the cache goes
        _case("evict-full", "evict", "float16", 32, 0, 8, 128, 8192, keep=4096, recent=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "write", "decode", "decode", "evict"])
    dtype = rng.choice(["float16", "bfloat16"])
    N_kv, group = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 7, 8])
    D = rng.choice([64, 128, 128, 128, 40, 80, 96])
    if kind == "prompt":
        N = min(32, N_kv * group) // N_kv * N_kv
        S = _log_int(rng, 16, 4096)
        prefix = _log_int(rng, 1, S) if rng.random() < 0.4 else 0
        B = _log_int(rng, 1, max(1, min(64, int(8 * 32 * 4096.0 ** 2 / (N * float(S) * (S + 2 * prefix))))))
        return _case(None, kind, dtype, B, N, N_kv, D, S, prefix=prefix)
    paged = rng.random() < 0.4
    most = {"write": 16 * 8 * 4096 * 128, "decode": 32 * 8 * 16384 * 128, "evict": 32 * 8 * 8192 * 128}[kind]
    S = _log_int(rng, 64, {"write": 8192, "decode": 32768, "evict": 16384}[kind])
    S = -(-S // PAGE) * PAGE if paged else S
    B = _log_int(rng, 1, max(1, min(64, most // (N_kv * S * D))))
    if kind == "write":
        return _case(None, kind, dtype, B, 0, N_kv, D, S, new=1 if rng.random() < 0.3 else _log_int(rng, 2, S), paged=paged)
    if kind == "decode":
        return _case(None, kind, dtype, B, N_kv * group, N_kv, D, S, weights=rng.random() < 0.5, paged=paged)
    keep = max(1, int(S * rng.uniform(0.1, 0.9)))
    return _case(None, kind, dtype, B, 0, N_kv, D, S, keep=keep, recent=int(keep * rng.uniform(0.0, 0.5)), paged=paged)


def _lengths(c):
    """Lengths of a batch's sequences, as they follow from its sizes: (rows there are before, rows that the call is about)."""
    r = random.Random("%d %d %d %d" % (c["B"], c["S"], c["new"], c["prefix"]))
    if c["kind"] == "prompt":
        rows = [c["S"]] + [_log_int(r, 1, c["S"]) if c["B"] <= 4 else r.randint(max(1, c["S"] // 4), c["S"]) for _ in range(c["B"] - 1)]
        return [r.randint(0, c["prefix"]) for _ in rows], rows
    if c["kind"] == "write":
        rows = [c["new"]] + [r.randint(max(1, c["new"] // 4), c["new"]) for _ in range(c["B"] - 1)]
        return [r.randint(0, c["S"] - n) for n in rows], rows
    return [0] * c["B"], [c["S"]] + [r.randint(max(1, c["S"] // 4), c["S"]) for _ in range(c["B"] - 1)]


def _row_bytes(D):
    """A row of one head in the cache: 4 bits a value, 16 bits of scale and of minimum per group."""
    return D / 2.0 + -(-D // GROUP) * 4.0


def work(case):
    c = case
    before, rows = _lengths(c)
    T, wide, narrow = sum(rows), 2.0 * c["D"], _row_bytes(c["D"])
    if c["kind"] == "prompt":
        keys = T + sum(before)
        pairs = sum(n * p + n * (n + 1) / 2.0 for p, n in zip(before, rows))
        return {"bytes": 2.0 * T * c["N"] * wide + 2.0 * keys * c["N_kv"] * wide, "flops": 4.0 * c["N"] * pairs * c["D"]}
    if c["kind"] == "write":             # 16 bits in, 4 bits out; and the way back
        return {"bytes": 2 * 2.0 * T * c["N_kv"] * (wide + narrow), "flops": 2.0 * 2 * T * c["N_kv"] * c["D"]}
    if c["kind"] == "decode":
        return {"bytes": 2.0 * c["B"] * c["N"] * wide + T * c["N_kv"] * (2.0 * narrow + (8.0 if c["weights"] else 0.0)),
                "flops": 4.0 * T * c["N"] * c["D"]}
    kept = sum(min(n, c["keep"]) for n in rows)
    # every probability; the kept rows in, out, and back as values; slots and probabilities of what is kept
    return {"bytes": 4.0 * T * c["N_kv"] + kept * c["N_kv"] * (2.0 * (3 * narrow + wide) + 8.0), "flops": 2.0 * kept * c["N_kv"] * c["D"]}


def _starts(rows):
    return torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda()


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _groups(x):
    """[..., D] -> [..., groups, 32]; a last group that is not full repeats its last value."""
    pad = -x.shape[-1] % GROUP
    if pad:
        x = torch.cat([x, x[..., -1:].expand(x.shape[:-1] + (pad,))], -1)
    return x.unflatten(-1, (-1, GROUP))


def _pack(x):
    """Codes, scales and minima of rows [..., D] in 16 bits."""
    dt, D = x.dtype, x.shape[-1]
    x = _groups(x.float())
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15.0).to(dt)
    above = s.float() > (hi - lo) / 15.0
    s = torch.where(above, (s.view(torch.int16) - above.short()).view(dt), s)      # the next lower 16-bit value
    inv = torch.where(s.float() > 0, 1.0 / s.float(), 0.0)
    codes = ((x - lo) * inv).round().clamp(0, 15).to(torch.uint8).flatten(-2)[..., :D].contiguous()
    return codes, s.squeeze(-1), lo.squeeze(-1).to(dt)


def _values(codes, s, m):
    D = codes.shape[-1]
    return (_groups(codes).float() * s.float().unsqueeze(-1) + m.float().unsqueeze(-1)).flatten(-2)[..., :D]


def _softmax(x):
    """Over the last dimension, in place; a row of -inf gives zeros."""
    m = x.amax(-1, keepdim=True)
    x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    return x.div_(x.sum(-1, keepdim=True).clamp_min_(1e-38))


def _plain_prompt(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    B, N, N_kv, D = c["B"], c["N"], c["N_kv"], c["D"]

    def padded(x, starts, most):
        at = starts[:-1, None].long() + torch.arange(most, device="cuda")
        return x[at.clamp_(max=x.shape[0] - 1)].transpose(1, 2).float()            # [B, heads, most, D]

    q = padded(s["q"], s["cu_q"], s["most_q"]).unflatten(1, (N_kv, N // N_kv))
    k, v = (padded(s[x], s["cu_k"], s["most_k"]).unsqueeze(2) for x in ("k", "v"))
    rows, keys = s["cu_q"].diff(), s["cu_k"].diff()
    i, j = torch.arange(s["most_q"], device="cuda"), torch.arange(s["most_k"], device="cuda")
    seen = j[None, None, :] <= (i[None, :, None] + (keys - rows)[:, None, None])
    p = torch.matmul(q * D ** -0.5, k.transpose(-1, -2)).masked_fill_(~seen[:, None, None], -math.inf)
    o = torch.matmul(_softmax(p), v).flatten(1, 2).transpose(1, 2)                 # [B, most, N, D]
    return o[i[None, :] < rows[:, None]].to(dt)


def _plain_write(s):
    dt = s["k"].dtype
    return tuple(_values(*_pack(s[x])).to(dt) for x in ("k", "v"))


def _plain_decode(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    B, N, N_kv, D = c["B"], c["N"], c["N_kv"], c["D"]
    q = s["q"].float().view(B, N_kv, N // N_kv, D) * D ** -0.5
    p = torch.matmul(q, _values(*s["k"]).transpose(-1, -2))                        # [B, N_kv, group, S]
    p.masked_fill_((torch.arange(c["S"], device="cuda") >= s["lens"][:, None])[:, None, None], -math.inf)
    p = _softmax(p)
    y = torch.matmul(p, _values(*s["v"])).view(B, N, 1, D).to(dt)
    return (y, s["weights"].add_(p.sum(2))) if c["weights"] else y


def _plain_evict(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    lens = s["lens"][:, None, None]
    i = torch.arange(c["S"], device="cuda")
    w = torch.where(i >= lens, -math.inf, torch.where(i >= lens - c["recent"], math.inf, s["weights"]))
    at = w.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    at = torch.where(at < lens, at, c["S"]).sort(dim=-1).values
    there = at < c["S"]
    kept = torch.where(there, at, -1).int()
    at = at.clamp_max(c["S"] - 1)
    weights = torch.where(there, s["weights"].gather(-1, at), 0.0)
    rows = there.transpose(1, 2)[..., 0]                                           # the same number in every head

    def take(pool):
        some = [x.gather(2, at[..., None].expand(at.shape + (x.shape[-1],))) for x in pool]
        return _values(*some).transpose(1, 2)[rows].to(dt)                         # [tokens, N_kv, D]

    return kept, weights, s["lens"].clamp(max=c["keep"]), take(s["k"]), take(s["v"])


# ---------------------------------------------------------------------------------------------------------------------
# a user's program
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    dt = DTYPES[c["dtype"]]
    B, N, N_kv, D, S = (c[k] for k in ("B", "N", "N_kv", "D", "S"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    before, rows = _lengths(c)
    T = sum(rows)

    def normal(*shape):
        return torch.empty(shape, device="cuda", dtype=dt).normal_(generator=g)

    def keys(*shape):
        """Keys as projections give them: some columns of a head are larger, and off zero."""
        x = normal(*shape)
        scale = torch.empty((N_kv, D), device="cuda").normal_(0.0, 0.5, generator=g).exp_()
        shift = torch.empty((N_kv, D), device="cuda").normal_(0.0, 0.5, generator=g)
        return x.mul_(scale.to(dt)).add_(shift.to(dt))

    s = {"case": c}
    if c["kind"] == "prompt":
        Tk = T + sum(before)
        s.update(q=normal(T, N, D), k=keys(Tk, N_kv, D), v=normal(Tk, N_kv, D), cu_q=_starts(rows),
                 cu_k=_starts([p + n for p, n in zip(before, rows)]), most_q=max(rows), most_k=max(p + n for p, n in zip(before, rows)))
        return s
    def cache(slots):
        """The cache object of this package, as a serving program makes it at its start."""
        from acctransformer_b200 import Kv4Cache
        if not c["paged"]:
            return Kv4Cache(B, N_kv, slots, D, dtype=dt)
        per = -(-slots // PAGE)
        order = torch.randperm(B * per, generator=torch.Generator().manual_seed(seed))      # pages come as they were free
        return Kv4Cache(B, N_kv, per * PAGE, D, dtype=dt, page_size=PAGE, block_table=order.int().view(B, per).cuda())

    if c["kind"] == "write":
        s.update(k=keys(T, N_kv, D), v=normal(T, N_kv, D), start=torch.tensor(before, dtype=torch.int32).cuda(), cu=_starts(rows))
        if own:
            s["cache"] = cache(S)
        return s
    if N:
        s["q"] = normal(B, N, 1, D)
    s["lens"] = torch.tensor(rows, dtype=torch.int32).cuda()
    if c["weights"] or c["kind"] == "evict":
        # heavy tails over the context; tokens that have only just come have none yet
        w = torch.empty((B, N_kv, S), device="cuda").normal_(-4.0, 1.5, generator=g).exp_()
        s["weights"] = w * (torch.arange(S, device="cuda") < s["lens"][:, None, None] - S // 16)
    k, v = keys(B, S, N_kv, D), normal(B, S, N_kv, D)
    if not own:      # in the place of the cache that the program has filled before: its content, as plain tensors
        s["k"], s["v"] = (tuple(x.transpose(1, 2).contiguous() for x in _pack(y)) for y in (k, v))
        return s
    s["cache"] = cache(S)
    s["cache"].append(k.flatten(0, 1), v.flatten(0, 1), torch.zeros(B, dtype=torch.int32, device="cuda"), _starts([S] * B))
    if c["kind"] == "decode":
        from acctransformer_b200 import Kv4Workspace
        s["workspace"] = Kv4Workspace(B, N, N_kv, S, D, "cuda", weights=c["weights"])      # kept by the serving loop
        return s
    kept = [min(n, c["keep"]) for n in rows]
    s.update(out=cache(c["keep"]), start=torch.zeros(B, dtype=torch.int32, device="cuda"), cu=_starts(kept), total=sum(kept))
    return s


def run(s):
    c = s["case"]
    if not own:
        return {"prompt": _plain_prompt, "write": _plain_write, "decode": _plain_decode, "evict": _plain_evict}[c["kind"]](s)
    if c["kind"] == "prompt":
        from acctransformer_b200 import flash_attention_packed
        return flash_attention_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=True)
    if c["kind"] == "write":
        s["cache"].append(s["k"], s["v"], s["start"], s["cu"])
        return s["cache"].read(s["start"], s["cu"], total=s["k"].shape[0])
    if c["kind"] == "decode":
        y = s["cache"].decode(s["q"], s["lens"], weights=s.get("weights"), workspace=s["workspace"])
        return (y, s["weights"]) if c["weights"] else y
    kept, weights, lens = s["cache"].evict(s["weights"], s["lens"], c["keep"], c["recent"], s["out"])
    k, v = s["out"].read(s["start"], s["cu"], total=s["total"])
    return kept, weights[..., :c["keep"]], lens, k, v


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    before, rows = _lengths(c)
    D, N_kv = c["D"], c["N_kv"]

    def attend(q, k, v, hidden):
        """q [heads, rows, D] on k, v [keys, D]; hidden [rows, keys]."""
        x = (q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
        p = (x - x.logsumexp(-1, keepdim=True)).exp()
        return p, p @ v

    if c["kind"] == "prompt":
        pairs = sum(n * (p + n) for p, n in zip(before, rows))
        if 4.0 * c["N"] * pairs * D > 4e13:
            return None
        outs, at_q, at_k = [], 0, 0
        for p, n in zip(before, rows):
            q, k, v = s["q"][at_q:at_q + n].double(), s["k"][at_k:at_k + p + n].double(), s["v"][at_k:at_k + p + n].double()
            hidden = torch.ones(n, p + n, dtype=torch.bool, device="cuda").triu_(p + 1)
            o = torch.empty_like(q)
            per = c["N"] // N_kv
            for h in range(N_kv):
                o[:, h * per:(h + 1) * per] = attend(q[:, h * per:(h + 1) * per].transpose(0, 1), k[:, h], v[:, h], hidden)[1].transpose(0, 1)
            outs.append(o)
            at_q, at_k = at_q + n, at_k + p + n
        return torch.cat(outs)

    if c["kind"] == "write":
        def through(x):
            dt, x = x.dtype, x.double()
            out = torch.empty_like(x)
            for at in range(0, D, GROUP):
                y = x[..., at:at + GROUP]
                m, top = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
                # the step, cut to the 11 or 8 leading bits of the type (no group here has one below its normal numbers)
                f, e = torch.frexp((top - m) / 15)
                bits = 11 if dt == torch.float16 else 8
                step = torch.ldexp(torch.floor(torch.ldexp(f, torch.tensor(bits, device="cuda"))), e - bits)
                c_ = torch.minimum(torch.round((y - m) / step.where(step > 0, 1.0)), torch.tensor(15.0, dtype=torch.float64, device="cuda"))
                out[..., at:at + GROUP] = m + step * c_
            return out
        return through(s["k"]), through(s["v"])

    def value(pool, b, h, at):
        """Rows `at` of one sequence's head, as the values they stand for."""
        codes, scale, low = (x[b, h][at].double() for x in pool)
        of = torch.arange(D, device="cuda") // GROUP
        return low[:, of] + codes * scale[:, of]

    if c["kind"] == "decode":
        per = c["N"] // N_kv
        y = torch.zeros(c["B"], c["N"], 1, D, dtype=torch.float64, device="cuda")
        w = s["weights"].double() if c["weights"] else None
        for b, n in enumerate(rows):
            for h in range(N_kv):
                k, v = (value(s[x], b, h, slice(0, n)) for x in ("k", "v"))
                q = s["q"][b, h * per:(h + 1) * per].double()
                p, o = attend(q, k, v, torch.zeros(1, n, dtype=torch.bool, device="cuda"))
                y[b, h * per:(h + 1) * per] = o
                if w is not None:
                    w[b, h, :n] += p.sum((0, 1))
        return y if w is None else (y, w)

    w_out = torch.zeros(c["B"], N_kv, c["keep"], dtype=torch.float64, device="cuda")
    ks, vs = [], []
    for b, n in enumerate(rows):
        m = min(n, c["keep"])
        k, v = (torch.empty(m, N_kv, D, dtype=torch.float64, device="cuda") for _ in range(2))
        for h in range(N_kv):
            old = max(0, n - c["recent"])
            w = s["weights"][b, h, :n].double()
            best = torch.argsort(-w[:old], stable=True)[:max(0, m - (n - old))]
            at = torch.cat([best.sort().values, torch.arange(old, n, device="cuda")])
            w_out[b, h, :m] = w[at]
            k[:, h], v[:, h] = value(s["k"], b, h, at), value(s["v"], b, h, at)
        ks.append(k)
        vs.append(v)
    return None, w_out, None, torch.cat(ks), torch.cat(vs)
