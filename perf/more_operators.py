"""Linear attention with a decay for each head, and rotary positions with several axes, as cases that can be timed: in plain
torch, or through this package's entry points.

* ``rotary``  queries and keys turned by their positions on one to three axes; ``grad``: and the way back of a training step;
* ``prompt``  linear attention over packed prompts of different lengths, with the state behind every prompt;
* ``train``   linear attention over a batch and the gradients of its queries, keys and values;
* ``step``    one token per sequence: the state moves on, and is read.

    S_t = exp(g) S_(t-1) + k_t v_t^T        y_t = scale S_t^T q_t        g <= 0 for each head, scale = D^-1/2
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
CHUNK = 128        # tokens that the plain form takes at a time
BASE = 10000.0


def _case(name, kind, dtype, B, N, N_kv, D, S, **more):
    c = {"kind": kind, "dtype": dtype, "B": B, "N": N, "N_kv": N_kv, "D": D, "S": S, "state": False, "padded": False,
         "axes": 1, "rotated": D, "adjacent": False, "per_axis": False, "grad": False, "far": 4096}
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the queries and keys of a decoding step, far into long contexts: nothing but launch and call
        _case("rotary-token", "rotary", "bfloat16", 16, 32, 8, 128, 1, far=131072),
        # patches of a few images, rows and columns, heads of an odd width of which a part is turned, neighbours as pairs
        _case("rotary-images", "rotary", "float16", 5, 16, 16, 80, 1801, axes=2, rotated=64, adjacent=True, per_axis=True, far=128),
        # a training batch of video tokens: time, height and width, there and back
        _case("rotary-video", "rotary", "bfloat16", 2, 32, 8, 128, 8192, axes=3, grad=True, far=1024),
        # a few chat turns that arrive together: latency, one or two tiles for each sequence and head
        _case("prompt-short", "prompt", "bfloat16", 4, 16, 16, 128, 200),
        # the next chunks of prompts whose states are there already: ragged, grouped narrow heads
        _case("prompt-chunks", "prompt", "float16", 24, 16, 4, 64, 1500, state=True),
        # long documents
        _case("prompt-long", "prompt", "bfloat16", 2, 32, 32, 128, 16384),
        # a small model's step
        _case("train-small", "train", "float16", 2, 8, 8, 64, 500),
        # a padded batch of odd sizes, grouped heads
        _case("train-odd", "train", "bfloat16", 3, 12, 4, 80, 1777, padded=True),
        # a full training batch
        _case("train-full", "train", "bfloat16", 4, 32, 32, 128, 4096),
        # a decoding step of a few interactive users
        _case("step-few", "step", "bfloat16", 4, 32, 32, 128, 1),
        # odd width, grouped heads
        _case("step-odd", "step", "float16", 7, 12, 3, 80, 1),
        # a decoding step of a full serving batch
        _case("step-full", "step", "bfloat16", 128, 32, 32, 128, 1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "prompt", "prompt", "train", "train", "step"])
    dtype = rng.choice(["float16", "bfloat16"])
    N_kv, group = rng.choice([1, 2, 4, 8, 12, 16, 32]), rng.choice([1, 1, 1, 2, 4])
    N = N_kv * (group if N_kv * group <= 32 else 1)
    D = rng.choice([64, 128, 128, 128, 40, 80, 96])
    if kind == "rotary":
        S = _log_int(rng, 1, 8192)
        B = _log_int(rng, 1, max(1, min(64, 2 * 8192 * 40 * 128 // (S * (N + N_kv) * D))))
        rotated = D if rng.random() < 0.7 else D // 2
        return _case(None, kind, dtype, B, N, N_kv, D, S, axes=rng.choice([1, 2, 3]), rotated=rotated, adjacent=rng.random() < 0.4,
                     per_axis=rng.random() < 0.4, grad=rng.random() < 0.4, far=_log_int(rng, 64, 1 << 20))
    if kind == "step":
        return _case(None, kind, dtype, _log_int(rng, 1, 128), N, N_kv, D, 1)
    S = _log_int(rng, 1 if kind == "prompt" else 16, 16384)
    most = 2 * 16384 * 32 * 128 if kind == "prompt" else 4 * 4096 * 32 * 128
    B = _log_int(rng, 1, max(1, min(64, most // (S * N * D))))
    return _case(None, kind, dtype, B, N, N_kv, D, S, state=kind == "prompt" and rng.random() < 0.5,
                 padded=kind == "train" and rng.random() < 0.3)


def _lengths(c):
    """Lengths of a batch's sequences, as they follow from its sizes."""
    r = random.Random("%d %d %d" % (c["B"], c["S"], c["D"]))
    if c["kind"] == "prompt" or c["padded"]:
        return [c["S"]] + [_log_int(r, 1, c["S"]) if c["B"] <= 4 else r.randint(max(1, c["S"] // 4), c["S"]) for _ in range(c["B"] - 1)]
    return [c["S"]] * c["B"]


def work(case):
    c = case
    T, D, N, N_kv = float(sum(_lengths(c))), c["D"], c["N"], c["N_kv"]
    row = 2.0 * D
    if c["kind"] == "rotary":        # in and out, 6 operations for each pair
        both = 2.0 if c["grad"] else 1.0
        return {"bytes": both * T * (2.0 * (N + N_kv) * row + 4.0 * c["axes"]), "flops": both * 3.0 * T * (N + N_kv) * c["rotated"]}
    state = 4.0 * c["B"] * N * D * D
    if c["kind"] == "step":          # every state in and out
        return {"bytes": 2.0 * state + T * (2 * N + 2 * N_kv) * row, "flops": 5.0 * T * N * D * D}
    if c["kind"] == "prompt":        # k v^T into the state, the state times q
        return {"bytes": T * (2 * N + 2 * N_kv) * row + state * (2.0 if c["state"] else 1.0), "flops": 4.0 * T * N * D * D}
    # there: q, k, v, y; back: q, k, v, dy in, three gradients out; the two states once each way, five products with them
    return {"bytes": T * (5 * N + 6 * N_kv) * row, "flops": 14.0 * T * N * D * D}


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _powers(g, n):
    """exp(g n) in 32 bits, g [N], n of any shape: [N, ...]."""
    return (g.double().view(-1, *[1] * n.dim()) * n.double()).exp().float()


def _linear(a, b, c, g, initial=None):
    """sum over i <= t of exp(g (t - i)) (a_t . b_i) c_i, all [B, N, S, D] in 32 bits, with an initial state [B, N, D, D]."""
    B, N, S, D = a.shape
    pad = -S % CHUNK
    a, b, c = (torch.nn.functional.pad(x, (0, 0, 0, pad)).unflatten(2, (-1, CHUNK)) for x in (a, b, c))
    chunks = a.shape[2]
    i = torch.arange(CHUNK, device=a.device)
    inside = torch.where(i[:, None] >= i, _powers(g, (i[:, None] - i).clamp_min(0)), 0.0)
    y = torch.matmul(torch.matmul(a, b.transpose(-1, -2)).mul_(inside[:, None]), c)
    states = torch.matmul((b * _powers(g, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2), c).flatten(-2)      # [B, N, chunks, D D]
    j = torch.arange(chunks, device=a.device)
    from_j = torch.where(j[:, None] > j, _powers(g, ((j[:, None] - 1 - j) * CHUNK).clamp_min(0)), 0.0)
    before = torch.matmul(from_j, states)
    if initial is not None:
        before = before + _powers(g, j * CHUNK)[..., None] * initial.flatten(-2)[:, :, None]
    before = before.unflatten(-1, (D, D))
    y += torch.matmul(a, before).mul_(_powers(g, i + 1)[:, None, :, None])
    return y.flatten(2, 3)[:, :, :S]


def _heads(x, N):
    return x.repeat_interleave(N // x.shape[1], 1) if x.shape[1] != N else x


def _plain_prompt(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    n = s["cu"].diff()
    i = torch.arange(c["S"], device="cuda")
    there = i < n[:, None]
    at = (s["cu"][:-1, None].long() + i).clamp_(max=s["q"].shape[0] - 1)
    q, k, v = (_heads((s[x][at].float() * there[..., None, None]).transpose(1, 2), c["N"]) for x in ("q", "k", "v"))
    y = _linear(q * c["D"] ** -0.5, k, v, s["g"], s.get("state"))
    left = (n[:, None] - 1 - i).clamp_min(0)                                        # tokens behind
    w = _powers(s["g"], left).transpose(0, 1)[..., None]                            # [B, N, S, 1]
    state = torch.matmul((k * w).transpose(-1, -2), v)
    if c["state"]:
        state = s["state"].mul_(_powers(s["g"], n).transpose(0, 1)[..., None, None]).add_(state)
    return y.transpose(1, 2)[there].to(dt), state


def _plain_train(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    B, N, N_kv, D, S = (c[x] for x in ("B", "N", "N_kv", "D", "S"))
    q, k, v, dy = (_heads(s[x].detach().float(), N) for x in ("q", "k", "v", "dy"))
    if c["padded"]:
        there = (torch.arange(S, device="cuda") < s["lens"][:, None])[:, None, :, None]
        q, k, v, dy = (x * there for x in (q, k, v, dy))
    q, dy = q, dy * D ** -0.5
    back = lambda x, y, z: _linear(x.flip(2), y.flip(2), z.flip(2), s["g"]).flip(2)  # noqa: E731
    shared = lambda x: x.unflatten(1, (N_kv, -1)).sum(2).to(dt)  # noqa: E731
    return (_linear(q * D ** -0.5, k, v, s["g"]).to(dt), _linear(dy, v, k, s["g"]).to(dt), shared(back(v, dy, q)), shared(back(k, q, dy)))


def _plain_step(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    q, k, v = (_heads(s[x].float(), c["N"]) for x in ("q", "k", "v"))               # [B, N, 1, D]
    s["state"].mul_(s["g"].double().exp().float()[:, None, None]).add_(k.transpose(-1, -2) * v)
    return torch.matmul(q * c["D"] ** -0.5, s["state"]).to(dt), s["state"]


def _pairs_of(c):
    """Of each pair that is turned: its axis, and its angle per position."""
    pairs, axes = c["rotated"] // 2, c["axes"]
    sections = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if c["per_axis"]:
        turn = [BASE ** (-i / n) for n in sections for i in range(n)]
    else:
        turn = [BASE ** (-i / pairs) for i in range(pairs)]
    return sections, axis, turn


def _plain_rotary(s):
    c, R = s["case"], s["case"]["rotated"]
    angle = s["positions"][s["axis"]].double() * s["turn"].view(-1, *[1] * (s["positions"].dim() - 1))        # [pairs, rows ...]
    cos, sin = (f(angle).float().movedim(0, -1).unsqueeze(1) for f in (torch.cos, torch.sin))                 # [rows ..., 1, pairs] or [B, 1, S, pairs]

    def turned(x, sin):
        y = x.detach().float()
        if c["adjacent"]:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            z = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([z, y[..., R:]], -1).to(x.dtype)

    out = turned(s["q"], sin), turned(s["k"], sin)
    return out + (turned(s["dq"], -sin), turned(s["dk"], -sin)) if c["grad"] else out


# ---------------------------------------------------------------------------------------------------------------------
# a user's program
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    dt = DTYPES[c["dtype"]]
    B, N, N_kv, D, S = (c[x] for x in ("B", "N", "N_kv", "D", "S"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = _lengths(c)
    T = sum(rows)

    def normal(*shape):
        return torch.empty(shape, device="cuda", dtype=dt).normal_(generator=g)

    def keys(*shape):
        """As projections give them: some columns are larger, and off zero."""
        x = normal(*shape)
        scale = torch.empty(D, device="cuda").normal_(0.0, 0.5, generator=g).exp_()
        shift = torch.empty(D, device="cuda").normal_(0.0, 0.3, generator=g)
        return x.mul_(scale.to(dt)).add_(shift.to(dt))

    s = {"case": c}
    if c["kind"] == "rotary":
        sections, axis, turn = _pairs_of(c)
        s.update(axis=torch.tensor(axis, device="cuda"), turn=torch.tensor(turn, dtype=torch.float64, device="cuda"))
        if c["grad"]:                # a batch of training: [B, heads, S, D]
            shapes, at = [(B, N, S, D), (B, N_kv, S, D)], (c["axes"], B, S)
        else:                        # packed rows: [T, heads, D]
            shapes, at = [(T, N, D), (T, N_kv, D)], (c["axes"], T)
        s["q"], s["k"] = normal(*shapes[0]), keys(*shapes[1])
        s["positions"] = torch.randint(0, c["far"], at, dtype=torch.int32, device="cuda", generator=g)
        if c["grad"]:
            s["dq"], s["dk"] = normal(*shapes[0]), normal(*shapes[1])
        if own:
            from acctransformer_b200 import Rotary
            s["rotary"] = Rotary(D, sections, base=BASE, adjacent=c["adjacent"], per_axis=c["per_axis"])
            if c["grad"]:
                s["q"].requires_grad_()
                s["k"].requires_grad_()
        return s
    # memories from two tokens to some hundreds, as the heads of one layer have them, and no two alike
    h = torch.arange(1, N + 1, device="cuda", dtype=torch.float32)
    s["g"] = -torch.exp2(-8.0 * h / N) * torch.empty(N, device="cuda").uniform_(0.5, 1.0, generator=g)
    if c["kind"] == "step":
        s.update(q=normal(B, N, 1, D), k=keys(B, N_kv, 1, D), v=normal(B, N_kv, 1, D),
                 state=torch.empty(B, N, D, D, device="cuda").normal_(0.0, 4.0, generator=g))
    elif c["kind"] == "prompt":
        s.update(q=normal(T, N, D), k=keys(T, N_kv, D), v=normal(T, N_kv, D),
                 cu=torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda())
        if c["state"]:
            s["state"] = torch.empty(B, N, D, D, device="cuda").normal_(0.0, 4.0, generator=g)
    else:
        s.update(q=normal(B, N, S, D).requires_grad_(), k=keys(B, N_kv, S, D).requires_grad_(), v=normal(B, N_kv, S, D).requires_grad_(),
                 dy=normal(B, N, S, D))
        if c["padded"]:
            s["lens"] = torch.tensor(rows, dtype=torch.int32).cuda()
    return s


def run(s):
    c = s["case"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "train": _plain_train, "step": _plain_step}[c["kind"]](s)
    if c["kind"] == "rotary":
        y = s["rotary"](s["q"], s["k"], s["positions"])
        return tuple(x.detach() for x in y) + torch.autograd.grad(y, (s["q"], s["k"]), (s["dq"], s["dk"])) if c["grad"] else y
    if c["kind"] == "prompt":
        from acctransformer_b200 import linear_attention_packed
        return linear_attention_packed(s["q"], s["k"], s["v"], s["g"], s["cu"], state=s.get("state"))
    if c["kind"] == "step":
        from acctransformer_b200 import linear_attention_step
        return linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"]), s["state"]
    from acctransformer_b200 import linear_attention
    y = linear_attention(s["q"], s["k"], s["v"], s["g"], seq_lens=s.get("lens"))
    return (y.detach(),) + torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dy"])


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, N, N_kv, D, S = (c[x] for x in ("B", "N", "N_kv", "D", "S"))

    if c["kind"] == "rotary":
        def turned(x, sign):
            out = x.detach().double().clone()
            first = [2 * i for i in range(c["rotated"] // 2)] if c["adjacent"] else list(range(c["rotated"] // 2))
            step = 1 if c["adjacent"] else c["rotated"] // 2
            z = torch.complex(out[..., first], out[..., [i + step for i in first]])
            angle = torch.stack([s["positions"][a].double() * t for a, t in zip(s["axis"].tolist(), s["turn"].tolist())], -1) * sign
            z = z * torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
            out[..., first], out[..., [i + step for i in first]] = z.real, z.imag
            return out
        y = turned(s["q"], 1.0), turned(s["k"], 1.0)
        return y + (turned(s["dq"], -1.0), turned(s["dk"], -1.0)) if c["grad"] else y

    decay = s["g"].double()
    per = N // N_kv

    def attend(q, k, v, state, step=256):
        """Sequences of one length, [B, N, n, D]: outputs, and the state behind them."""
        outs = []
        for at in range(0, q.shape[2], step):
            x, y, z = (t[:, :, at:at + step] for t in (q, k, v))
            n = x.shape[2]
            i = torch.arange(n, device="cuda", dtype=torch.float64)
            apart = (i[:, None] - i).tril_()
            p = x @ y.transpose(-1, -2) * torch.exp(decay[:, None, None] * apart).tril()
            outs.append(p @ z + torch.exp(decay[:, None] * (i + 1))[..., None] * (x @ state))
            state = torch.exp(decay * n)[:, None, None] * state + (y * torch.exp(decay[:, None] * (n - 1 - i))[..., None]).transpose(-1, -2) @ z
        return torch.cat(outs, 2), state

    def shared(x):
        return x.repeat_interleave(per, 1)

    if c["kind"] == "step":
        q, k, v = s["q"].double() / math.sqrt(D), shared(s["k"].double()), shared(s["v"].double())
        state = torch.exp(decay)[:, None, None] * s["state"].double() + k.transpose(-1, -2) @ v
        return q @ state, state

    if c["kind"] == "prompt":
        ys, states, at = [], [], 0
        for b, n in enumerate(_lengths(c)):
            q, k, v = (s[x][at:at + n].double().transpose(0, 1).unsqueeze(0) for x in ("q", "k", "v"))
            start = s["state"][b:b + 1].double() if c["state"] else torch.zeros(1, N, D, D, dtype=torch.float64, device="cuda")
            y, state = attend(q / math.sqrt(D), shared(k), shared(v), start)
            ys.append(y[0].transpose(0, 1))
            states.append(state)
            at += n
        return torch.cat(ys), torch.cat(states)

    out = [torch.zeros(B, heads, S, D, dtype=torch.float64, device="cuda") for heads in (N, N, N_kv, N_kv)]
    for b, n in enumerate(_lengths(c)):      # one at a time: the graph of the backward is large
        leaves = [s[x][b:b + 1, :, :n].detach().double().requires_grad_() for x in ("q", "k", "v")]
        zero = torch.zeros(1, N, D, D, dtype=torch.float64, device="cuda")
        y, _ = attend(leaves[0] / math.sqrt(D), shared(leaves[1]), shared(leaves[2]), zero)
        grads = torch.autograd.grad(y, leaves, s["dy"][b:b + 1, :, :n].double())
        for o, x in zip(out, (y.detach(),) + grads):
            o[b, :, :n] = x[0]
    return tuple(out)
