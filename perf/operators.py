"""What a host asks of the row and norm operators around the experts: cases, plain forms, 64-bit values.

  dispatch       tokens' rows sorted by expert: positions, offsets, counts and the rows themselves
  dispatch_grad  the gradient of the tokens (and of the routing weights, where they scale the rows)
  collect        the rows back at their tokens: a weighted sum, beside what the shared expert gave
  collect_grad   the gradient of the rows and of the routing weights
  norm           a block's output normed, gated and added to the scaled residual stream, which is normed for the
                 next block
  norm_grad      the gradient of all of that: streams, norm weights, gate

Shapes are those of `pelica_b200.synth`'s configurations or of the same kind. Routing is top-k of logits with an uneven
popularity of the experts; `masked` tokens are the padding of a batch (their pairs have no row).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # one token of a decode step, one layer of 64 experts
        dict(name="dispatch_decode_1", op="dispatch", dtype="f32", tokens=1, d=2048, top_k=8, experts=64),
        # a padded batch of prompts in front of grouped products with tiles of 16 rows
        dict(name="dispatch_prompt_4096", op="dispatch", dtype="bf16", tokens=4096, d=7168, top_k=8, experts=256, align=16,
             masked=0.05),
        # training with the routing weight on the way in
        dict(name="dispatch_grad_2048", op="dispatch_grad", dtype="f32", tokens=2048, d=2048, top_k=8, experts=128, scale=True),
        # a ragged batch on a rank that holds a quarter of the experts
        dict(name="dispatch_grad_shard_3001", op="dispatch_grad", dtype="bf16", tokens=3001, d=2880, top_k=4, experts=32,
             first=8, local=8),
        # eight sequences decoded together, the shared expert's output beside the routed ones
        dict(name="collect_decode_8", op="collect", dtype="f32", tokens=8, d=7168, top_k=8, experts=256, add=True),
        # a prompt chunk
        dict(name="collect_prompt_4096", op="collect", dtype="bf16", tokens=4096, d=2048, top_k=8, experts=128, align=128),
        # a training batch, groups padded to the products' tiles
        dict(name="collect_grad_8192", op="collect_grad", dtype="bf16", tokens=8192, d=2048, top_k=8, experts=128, align=128),
        # widths that no vector divides, rows inside a wider buffer
        dict(name="collect_grad_odd_333", op="collect_grad", dtype="f16", tokens=333, d=1001, top_k=5, experts=40, pitch=3),
        # one token between two blocks with norms on both sides
        dict(name="norm_decode_1", op="norm", dtype="f32", tokens=1, d=7168, post=True, pre=True),
        # a large prompt, a gate for each token
        dict(name="norm_prompt_16384", op="norm", dtype="bf16", tokens=16384, d=2048, post=True, pre=True, gate="token"),
        # a training batch of a wide model, a learned gate for each channel
        dict(name="norm_grad_4096", op="norm_grad", dtype="bf16", tokens=4096, d=7168, post=True, pre=True, gate="channel"),
        # a pre-norm model with a scaled residual stream, weights stored as w - 1
        dict(name="norm_grad_777", op="norm_grad", dtype="f32", tokens=777, d=2880, post=False, pre=True, alpha=0.5, offset=1.0),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["dispatch", "dispatch_grad", "collect", "collect_grad", "norm", "norm_grad"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))
    unit = rng.choice([1, 8, 64, 256])
    d = max(unit, _spread(rng, 64, 8192) // unit * unit)
    case.update(d=d, tokens=_spread(rng, 1, 16384), pitch=rng.choice([0, 0, 0, 8, 3]))
    if op.startswith("norm"):
        post = rng.random() < 0.7
        case.update(post=post, pre=not post or rng.random() < 0.8, gate=rng.choice(["none", "channel", "token"]),
                    alpha=rng.choice([1.0, 0.5, 1.25]), beta=rng.choice([1.0, 0.22]), offset=rng.choice([0.0, 1.0]),
                    wtype=rng.choice(["f32", case["dtype"]]))
        most = 85_000_000 // (d * SIZE[case["dtype"]])
    else:
        experts = _spread(rng, 4, 512)
        case.update(experts=experts, top_k=rng.randint(1, min(10, experts)), align=rng.choice([1, 1, 16, 128]),
                    masked=rng.choice([0.0, 0.0, 0.1]))
        if rng.random() < 0.25 and experts >= 8:
            case.update(local=experts // 4, first=rng.randrange(4) * (experts // 4))
        if op.startswith("dispatch"):
            case["scale"] = rng.random() < 0.5
        elif op == "collect":
            case["add"] = rng.random() < 0.5
        # rows read and written, the padding of every group among them
        row = d * SIZE[case["dtype"]]
        most = (240_000_000 // row - experts * (case["align"] - 1) // 2) // case["top_k"]
    case["tokens"] = max(1, min(case["tokens"], most))
    return case


# --------------------------------------------------------------------------
# states
# --------------------------------------------------------------------------
class State:
    pass


def _plan(ids, s):
    """Stable counting sort of the pairs by expert: offset, count, pos, row_pair; all int32, -1 = none."""
    flat = ids.reshape(-1).long() - s.first
    local = (flat >= 0) & (flat < s.local) & (ids.reshape(-1) >= 0)
    key = torch.where(local, flat, s.local)
    order = torch.argsort(key, stable=True)
    count = torch.zeros(s.local + 1, dtype=torch.long, device=key.device).scatter_add_(0, key, torch.ones_like(key))[:s.local]
    padded = (count + s.align - 1) // s.align * s.align
    offset = torch.cat([padded.new_zeros(1), padded.cumsum(0)])
    begin = torch.cat([count.new_zeros(1), count.cumsum(0)])  # without padding
    rank = torch.empty_like(order)
    rank[order] = torch.arange(order.numel(), device=order.device)
    pos = torch.where(local, rank - begin[key] + offset[key], -1)
    row_pair = torch.full((s.max_rows + 1,), -1, device=pos.device)
    row_pair[torch.where(local, pos, s.max_rows)] = torch.arange(pos.numel(), device=pos.device)
    return offset.int(), count.int(), pos.int().reshape(ids.shape), row_pair[:-1].int()


def _wide(t, pitch):
    """The rows of t inside a buffer that is `pitch` columns wider."""
    if not pitch:
        return t
    b = torch.zeros(t.shape[0], t.shape[1] + pitch, dtype=t.dtype, device=t.device)
    b[:, :t.shape[1]] = t
    return b[:, :t.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    s = State()
    s.case, s.op = case, case["op"]
    s.dtype, s.T, s.d = TYPES[case["dtype"]], case["tokens"], case["d"]
    s.pitch = case.get("pitch", 0)
    s.handle = None

    def normal(rows, sigma=1.0, cols=s.d):
        return _wide((torch.randn(rows, cols, device="cuda", generator=g) * sigma).to(s.dtype), s.pitch)

    def empty(rows):
        return _wide(torch.zeros(rows, s.d, dtype=s.dtype, device="cuda"), s.pitch)

    if s.op.startswith("norm"):
        s.post, s.pre, s.gate = case["post"], case["pre"], case.get("gate", "none")
        s.alpha, s.beta, s.offset = case.get("alpha", 1.0), case.get("beta", 1.0), case.get("offset", 0.0)
        wtype = TYPES[case.get("wtype", "f32")]

        def weights(n, mean, sigma):
            return (torch.randn(n, device="cuda", generator=g) * sigma + mean).to(wtype)

        s.w_post = weights(s.d, 1.0 - s.offset, 0.2) if s.post else None
        s.w_pre = weights(s.d, 1.0 - s.offset, 0.2) if s.pre else None
        s.g = None if s.gate == "none" else weights(s.d if s.gate == "channel" else s.T, 0.3, 0.3)
        # a residual stream with a few channels far above the others, as trained ones have them
        loud = 1.0 + 30.0 * (torch.rand(s.d, device="cuda", generator=g) < 0.002).float()
        s.x, s.f = normal(s.T), normal(s.T, 0.5)
        s.x.mul_(loud)  # in norm_grad: the stream behind the block
        s.r, s.n = empty(s.T), empty(s.T) if s.pre else None
        if s.op == "norm_grad":
            s.dr, s.dn = normal(s.T, 0.1), normal(s.T, 0.1) if s.pre else None
            s.df = empty(s.T)
            s.dx = s.r
            one = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
            s.dw_post, s.dw_pre = one(s.d) if s.post else None, one(s.d) if s.pre else None
            s.dg = None if s.g is None else one(s.g.numel())
        return s

    s.K, s.E = case["top_k"], case["experts"]
    s.first, s.local = case.get("first", 0), case.get("local", case["experts"])
    s.align, s.scale = case.get("align", 1), case.get("scale", False)
    pairs = s.T * s.K
    s.max_rows = pairs + min(s.local, pairs) * (s.align - 1)
    logits = torch.randn(s.T, s.E, device="cuda", generator=g) + 1.5 * torch.randn(s.E, device="cuda", generator=g)
    top, ids = torch.topk(logits, s.K, dim=1)
    ids[torch.rand(s.T, device="cuda", generator=g) < case.get("masked", 0.0)] = -1
    s.ids, s.w = ids.int(), torch.softmax(top, 1)
    # what the dispatch before made, for the calls behind it
    s.offset, s.count, s.pos, s.row_pair = _plan(s.ids, s)
    if s.op == "dispatch":
        s.x, s.rows = normal(s.T), empty(s.max_rows)
        s.offset, s.count, s.pos, s.row_pair = (torch.full_like(t, -1) for t in (s.offset, s.count, s.pos, s.row_pair))
        return s
    s.dw = torch.zeros(s.T, s.K, device="cuda")
    if s.op == "dispatch_grad":
        s.x, s.rows, s.y = normal(s.T) if s.scale else None, normal(s.max_rows), empty(s.T)
    elif s.op == "collect":
        s.rows, s.y = normal(s.max_rows), empty(s.T)
        s.add = normal(s.T) if case.get("add") else None
    else:
        s.rows, s.x, s.drows = normal(s.max_rows), normal(s.T), empty(s.max_rows)  # x: dy
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"dispatch": _dispatch, "dispatch_grad": _dispatch_grad, "collect": _collect, "collect_grad": _collect_grad,
            "norm": _norm, "norm_grad": _norm_grad}[s.op](s)


def _gathered(s):
    """[T][K][d] f32: the rows of the tokens' pairs, zero where a pair has none."""
    return s.rows[s.pos.clamp(min=0).long()].float() * (s.pos >= 0)[..., None]


def _dispatch(s):
    offset, count, pos, row_pair = _plan(s.ids, s)
    pair = row_pair.clamp(min=0).long()
    rows = s.x[pair // s.K].float()
    if s.scale:
        rows = rows * s.w.reshape(-1)[pair][:, None]
    rows = torch.where((row_pair >= 0)[:, None], rows, 0.0).to(s.dtype)
    return dict(offset=offset, count=count, pos=pos, row_pair=row_pair, rows=rows)


def _dispatch_grad(s):
    rows = _gathered(s)
    if not s.scale:
        return dict(dx=rows.sum(1).to(s.dtype))
    return dict(dx=(rows * s.w[..., None]).sum(1).to(s.dtype), dw=(rows * s.x.float()[:, None]).sum(-1))


def _collect(s):
    y = (_gathered(s) * s.w[..., None]).sum(1)
    if s.add is not None:
        y = y + s.add.float()
    return dict(y=y.to(s.dtype))


def _collect_grad(s):
    pair = s.row_pair.clamp(min=0).long()
    scale = torch.where(s.row_pair >= 0, s.w.reshape(-1)[pair], 0.0)
    drows = (s.x[pair // s.K].float() * scale[:, None]).to(s.dtype)
    return dict(drows=drows, dw=(_gathered(s) * s.x.float()[:, None]).sum(-1))


def _norm(s):
    x, p = s.x.float(), s.f.float()
    if s.post:
        p = p * torch.rsqrt(p.square().mean(-1, keepdim=True) + EPS) * (s.offset + s.w_post.float())
    if s.g is not None:
        p = p * (s.g.float() if s.gate == "channel" else s.g.float()[:, None])
    r = s.alpha * x + s.beta * p
    out = dict(r=r.to(s.dtype))
    if s.pre:
        out["n"] = (r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * (s.offset + s.w_pre.float())).to(s.dtype)
    return out


def _norm_grad(s):
    r, f, total = s.x.float(), s.f.float(), s.dr.float()
    out = {}
    if s.pre:
        dn = s.dn.float()
        rstd = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
        h = r * rstd
        u = dn * (s.offset + s.w_pre.float())
        total = total + rstd * (u - h * (u * h).mean(-1, keepdim=True))
        out["dw_pre"] = (dn * h).sum(0)
    out["dx"] = (s.alpha * total).to(s.dtype)
    k = p = f
    if s.post:
        rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
        k = f * rstd
        p = k * (s.offset + s.w_post.float())
    q = s.beta * total
    if s.g is not None:
        out["dg"] = (q * p).sum(0) if s.gate == "channel" else (q * p).sum(1)
        q = q * (s.g.float() if s.gate == "channel" else s.g.float()[:, None])
    if s.post:
        out["dw_post"] = (q * k).sum(0)
        v = q * (s.offset + s.w_post.float())
        q = rstd * (v - k * (v * k).mean(-1, keepdim=True))
    out["df"] = q.to(s.dtype)
    return out


_context = None


def _ctx():
    """The process's context, ordered on torch's stream, as a program beside torch has it."""
    global _context
    if _context is None:
        import pelica_b200 as pb

        _context = pb.Context(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream)
    return _context


def _at(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    import pelica_b200 as pb

    pitch = s.d + s.pitch
    if s.op.startswith("norm"):
        if s.handle is None:
            s.handle = pb.BlockNorm(_ctx(), s.d, dtype=s.case["dtype"], wtype=s.case.get("wtype", "f32"), post=s.post, pre=s.pre,
                                    gate=s.gate, alpha=s.alpha, beta=s.beta, eps_post=EPS, eps_pre=EPS, offset_post=s.offset,
                                    offset_pre=s.offset, stride=pitch)
            if s.op == "norm_grad":
                s.scratch = torch.empty(s.handle.scratch_bytes(s.T), dtype=torch.uint8, device="cuda")
        if s.op == "norm":
            s.handle.forward(s.T, _at(s.x), _at(s.f), _at(s.r), _at(s.n), w_post=_at(s.w_post), gate=_at(s.g), w_pre=_at(s.w_pre))
            return dict(r=s.r, n=s.n) if s.pre else dict(r=s.r)
        s.handle.grad(s.T, _at(s.x), _at(s.f), _at(s.dr), _at(s.dn), _at(s.dx), _at(s.df), w_post=_at(s.w_post), gate=_at(s.g),
                      w_pre=_at(s.w_pre), dw_post=_at(s.dw_post), dgate=_at(s.dg), dw_pre=_at(s.dw_pre), scratch=_at(s.scratch),
                      scratch_bytes=s.scratch.numel())
        out = dict(dx=s.dx, df=s.df, dw_pre=s.dw_pre, dw_post=s.dw_post, dg=s.dg)
        return {k: v for k, v in out.items() if v is not None}
    if s.handle is None:
        s.handle = pb.Rows(_ctx(), s.d, s.K, s.E, dtype=s.case["dtype"], first_expert=s.first, n_local=s.local, align=s.align,
                           x_stride=pitch, rows_stride=pitch)
        s.plan = s.handle.plan(s.max_rows, offset=_at(s.offset), count=_at(s.count), pos=_at(s.pos), row_pair=_at(s.row_pair))
    if s.op == "dispatch":
        s.handle.dispatch(s.T, _at(s.ids), s.plan, _at(s.x), _at(s.rows), w=_at(s.w) if s.scale else None)
        return dict(offset=s.offset, count=s.count, pos=s.pos, row_pair=s.row_pair, rows=s.rows)
    if s.op == "dispatch_grad":
        if not s.scale:
            s.handle.dispatch_grad(s.T, s.plan, _at(s.rows), _at(s.y))
            return dict(dx=s.y)
        s.handle.dispatch_grad(s.T, s.plan, _at(s.rows), _at(s.y), w=_at(s.w), x=_at(s.x), dw=_at(s.dw))
        return dict(dx=s.y, dw=s.dw)
    if s.op == "collect":
        s.handle.collect(s.T, s.plan, _at(s.rows), _at(s.y), w=_at(s.w), add=_at(s.add))
        return dict(y=s.y)
    s.handle.collect_grad(s.T, s.plan, _at(s.x), _at(s.drows), w=_at(s.w), rows=_at(s.rows), dw=_at(s.dw))
    return dict(drows=s.drows, dw=s.dw)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "norm":
        r = s.alpha * s.x.double()
        for t0 in range(0, s.T, 1024):
            at = slice(t0, min(s.T, t0 + 1024))
            f = s.f[at].double()
            if s.post:
                f = f / (f.pow(2).sum(1, keepdim=True) / s.d + EPS).sqrt() * (s.w_post.double() + s.offset)
            if s.gate == "channel":
                f = f * s.g.double()
            if s.gate == "token":
                f = f * s.g[at].double().unsqueeze(1)
            r[at] += s.beta * f
        if not s.pre:
            return dict(r=r)
        return dict(r=r, n=r / (r.pow(2).sum(1, keepdim=True) / s.d + EPS).sqrt() * (s.w_pre.double() + s.offset))
    if s.op == "norm_grad":
        return _exact_norm_grad(s)
    ids, none = s.ids.cpu().tolist(), -1
    lists = [[] for _ in range(s.local)]
    for t, chosen in enumerate(ids):
        for k, e in enumerate(chosen):
            if e >= 0 and s.first <= e < s.first + s.local:
                lists[e - s.first].append(t * s.K + k)
    pos, row_pair, offset, at = [none] * (s.T * s.K), [none] * s.max_rows, [0], 0
    for pairs in lists:
        for i, p in enumerate(pairs):
            pos[p], row_pair[at + i] = at + i, p
        at += math.ceil(len(pairs) / s.align) * s.align
        offset.append(at)
    used = torch.tensor([p for p in pos if p != none], dtype=torch.long, device="cuda")  # in the order of the pairs
    pair = torch.tensor([i for i, p in enumerate(pos) if p != none], dtype=torch.long, device="cuda")
    token, w = pair // s.K, s.w.double().reshape(-1)[pair].unsqueeze(1)
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if s.op == "dispatch":
        rows = torch.zeros(s.max_rows, s.d, dtype=torch.float64, device="cuda")
        rows[used] = s.x.double()[token] * (w if s.scale else 1.0)
        return dict(offset=whole(offset), count=whole([len(p) for p in lists]), pos=whole(pos).reshape(s.T, s.K),
                    row_pair=whole(row_pair), rows=rows)
    taken = s.rows[used].double()
    dw = torch.zeros(s.T * s.K, dtype=torch.float64, device="cuda")
    if s.op == "dispatch_grad":
        dx = torch.zeros(s.T, s.d, dtype=torch.float64, device="cuda").index_add_(0, token, taken * (w if s.scale else 1.0))
        if not s.scale:
            return dict(dx=dx)
        dw[pair] = torch.linalg.vecdot(taken, s.x.double()[token])
        return dict(dx=dx, dw=dw.reshape(s.T, s.K))
    if s.op == "collect":
        y = torch.zeros(s.T, s.d, dtype=torch.float64, device="cuda") if s.add is None else s.add.double()
        return dict(y=y.index_add_(0, token, taken * w))
    drows = torch.zeros(s.max_rows, s.d, dtype=torch.float64, device="cuda")
    drows[used] = s.x.double()[token] * w
    dw[pair] = torch.linalg.vecdot(taken, s.x.double()[token])
    return dict(drows=drows, dw=dw.reshape(s.T, s.K))


def _exact_norm_grad(s):
    """In slices of rows, from the quotient rule: d(v / m) = dv / m - v (v . dv) / (d m^3), m = sqrt(mean v^2 + eps)."""
    dx = torch.empty(s.T, s.d, dtype=torch.float64, device="cuda")
    df = torch.empty_like(dx)
    sums = {k: torch.zeros(s.d, dtype=torch.float64, device="cuda") for k in ("pre", "post", "gate")}
    by_token = torch.zeros(s.T, dtype=torch.float64, device="cuda")
    for t0 in range(0, s.T, 1024):
        at = slice(t0, min(s.T, t0 + 1024))
        r, f, total = s.x[at].double(), s.f[at].double(), s.dr[at].double()
        if s.pre:
            m = (r.pow(2).sum(1, keepdim=True) / s.d + EPS).sqrt()
            dn = s.dn[at].double()
            a = dn * (s.w_pre.double() + s.offset)
            total = total + a / m - r * (r * a).sum(1, keepdim=True) / (s.d * m.pow(3))
            sums["pre"] += (dn * r / m).sum(0)
        dx[at] = total * s.alpha
        m = (f.pow(2).sum(1, keepdim=True) / s.d + EPS).sqrt()
        weight = s.w_post.double() + s.offset if s.post else 1.0
        p = f / m * weight if s.post else f
        back = total * s.beta
        if s.gate == "channel":
            sums["gate"] += (back * p).sum(0)
            back = back * s.g.double()
        if s.gate == "token":
            by_token[at] = (back * p).sum(1)
            back = back * s.g[at].double().unsqueeze(1)
        if s.post:
            sums["post"] += (back * f / m).sum(0)
            a = back * weight
            back = a / m - f * (f * a).sum(1, keepdim=True) / (s.d * m.pow(3))
        df[at] = back
    out = dict(dx=dx, df=df)
    if s.pre:
        out["dw_pre"] = sums["pre"]
    if s.post:
        out["dw_post"] = sums["post"]
    if s.g is not None:
        out["dg"] = sums["gate"] if s.gate == "channel" else by_token
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    T, d, size = case["tokens"], case["d"], SIZE[case["dtype"]]
    row, op = d * size, case["op"]
    if op.startswith("norm"):
        wsize = SIZE[case.get("wtype", "f32")]
        vectors = int(case["post"]) + int(case["pre"]) + int(case.get("gate", "none") == "channel")
        if op == "norm":
            return {"bytes": float(T * row * (3 + int(case["pre"])) + vectors * d * wsize), "flops": 10.0 * T * d}
        return {"bytes": float(T * row * (5 + int(case["pre"])) + vectors * d * (wsize + 4)), "flops": 24.0 * T * d}
    K, E = case["top_k"], case["experts"]
    pairs = T * K * case.get("local", E) / E * (1.0 - case.get("masked", 0.0))
    align = case.get("align", 1)
    padding = min(case.get("local", E), pairs) * (align - 1) / 2  # half a tile a group that has rows
    index = 8.0 * T * K
    if op == "dispatch":
        return {"bytes": T * row + (pairs + padding) * row + index, "flops": pairs * d if case.get("scale") else 0.0}
    if op == "dispatch_grad":
        dw = bool(case.get("scale"))
        return {"bytes": pairs * row + (1 + dw) * T * row + index, "flops": (3.0 if dw else 1.0) * pairs * d}
    if op == "collect":
        return {"bytes": pairs * row + (1 + bool(case.get("add"))) * T * row + index, "flops": 2.0 * pairs * d}
    return {"bytes": T * row + (2 * pairs + padding) * row + index, "flops": 3.0 * pairs * d}
