"""The operators of a serving loop whose speed is kept in view: a paged k/v
cache (f16 or MXFP4) with what writes and reads it, and log probabilities.

    append     the rows of a batch: biases, per-head norms of q and k, the
               position rotation, k and v into the cache (mh_kv_append_dev),
               and the stored values read back (mh_kv_read_dev)
    attention  the rows of a batch over their sequences' pages
               (mh_kv_attention_dev): one token each, a few, or a prompt chunk
    logprobs   given tokens' log probabilities, the entropy and the most
               probable tokens of each row of logits (mh_logprobs_dev)

Head layouts are those of the models the framework serves (64 query heads on
8 of 64; 32 on 8 and 32 on 4 of 128) and generic ones. k and v are normal
values through the cache's own encoding, pages lie in random order.
"""
import math

import torch

own = False

EPS = 1e-5
F16, MXFP4 = 0, 1       # cache types, as MH_KV_F16 and MH_KV_MXFP4


# ------------------------------------------------------------------ cases

def _heads(nh, nkv, hd):
    return dict(nh=nh, nkv=nkv, hd=hd)


_A, _B, _C = _heads(64, 8, 64), _heads(32, 8, 128), _heads(32, 4, 128)


def _kv(kind, heads, dt, seqs, rows, lo, hi, page=64, window=0, sink=False, norm=False, name=None):
    """`seqs` sequences of lo..hi tokens (evenly spread over the logarithm), the last `rows` of each new."""
    c = dict(kind=kind, dt=dt, seqs=seqs, rows=rows, lo=lo, hi=hi, page=page, **heads)
    c.update(dict(window=window, sink=sink) if kind == "attention" else dict(norm=norm))
    return dict(c, name=name) if name else c


def listed():
    return [
        # the next token of one chat: the smallest append
        _kv("append", _A, "mxfp4", 1, 1, 1044, 1044, name="append_b1"),
        # a serving batch's next tokens, with norms of q and k
        _kv("append", _C, "f16", 64, 1, 17, 9000, norm=True, page=16, name="append_b64"),
        # three prompts of odd lengths
        _kv("append", _A, "mxfp4", 3, 667, 667, 4001, name="append_prompts"),
        # one chat's next token at a usual and at a very long context
        _kv("attention", _A, "mxfp4", 1, 1, 4100, 4100, sink=True, name="attend_b1_4k"),
        _kv("attention", _A, "mxfp4", 1, 1, 131071, 131071, sink=True, name="attend_b1_128k"),
        # a serving batch with contexts of all lengths
        _kv("attention", _A, "mxfp4", 32, 1, 100, 16000, sink=True, name="attend_b32"),
        # the same from an f16 cache, wider heads
        _kv("attention", _B, "f16", 16, 1, 500, 8191, page=16, name="attend_b16_f16"),
        # a sliding layer and a full layer of a long prompt
        _kv("attention", _A, "mxfp4", 1, 2000, 2000, 2000, window=128, sink=True, name="prompt_2000_window"),
        _kv("attention", _A, "mxfp4", 1, 4000, 4000, 4000, sink=True, name="prompt_4000"),
        # a chunk of a prompt behind a long context
        _kv("attention", _C, "f16", 1, 512, 16000, 16000, page=128, name="chunk_512_f16"),
        # the probability of a sampled token with its alternatives
        dict(name="logprobs_1", kind="logprobs", n=1, vocab=201088, ids=1, top=20, spread=4.0),
        # a prompt's tokens scored
        dict(name="logprobs_400", kind="logprobs", n=400, vocab=201088, ids=1, top=5, spread=4.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LAYOUTS = [_A, _A, _B, _C, _heads(16, 16, 64), _heads(24, 2, 96), _heads(8, 1, 256), _heads(40, 10, 32), _heads(12, 4, 192)]


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "prompt", "prompt", "logprobs", "logprobs"])
    if kind == "logprobs":
        return dict(kind=kind, n=_log(rng, 1, 400), vocab=_log(rng, 1000, 201088), ids=rng.randint(0, 4), top=rng.choice([0, 1, 5, 20, 32]),
                    spread=rng.choice([0.5, 2.0, 4.0, 10.0]))
    heads, dt = rng.choice(_LAYOUTS), rng.choice(["mxfp4", "mxfp4", "f16"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        seqs = _log(rng, 1, 64)
        rows = rng.choice([1, _log(rng, 1, max(1, 2000 // seqs))])
        lo = rows + _log(rng, 1, 2000)
        return _kv(kind, heads, dt, seqs, rows, lo, lo + rng.choice([0, _log(rng, 1, 4000)]), page, norm=rng.choice([False, True]))
    window, sink = rng.choice([0, 0, 128, 1000]), rng.choice([False, True])
    if kind == "attention":
        seqs, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 8])
        lo = rows + _log(rng, 1, 400000 // seqs // heads["nkv"])
        return _kv(kind, heads, dt, seqs, rows, lo, lo + rng.choice([0, lo]), page, window, sink)
    seqs = rng.choice([1, 1, 2, 5])
    rows = _log(rng, 16, 1500 // seqs)
    lo = rows + rng.choice([0, 0, _log(rng, 1, 8000 // seqs)])
    return _kv("attention", heads, dt, seqs, rows, lo, lo + rng.choice([0, 77]), page, window, sink)


def _seqs(c):
    """[(tokens, new rows)] of a batch; prompts of one batch differ in length a little."""
    n, out = c["seqs"], []
    for i in range(n):
        length = int(round(c["lo"] * (c["hi"] / c["lo"]) ** (i / (n - 1)))) if n > 1 else c["lo"]
        rows = max(1, c["rows"] - (i * 37) % 50) if c["rows"] > 100 else c["rows"]
        out.append((length, rows))
    return out


# ------------------------------------------------------------------ inputs

class _State:
    pass


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(shape, g, std=1.0, mean=0.0):
    return torch.randn(shape, device="cuda", generator=g) * std + mean


def _encode(x):
    """f32 x[..., hd] as MXFP4: (codes [..., hd / 2], exponent bytes [..., hd / 32])."""
    b = x.unflatten(-1, (-1, 32))
    f, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(f <= 0.875, e - 3, e - 2).clamp(-13, 13)
    a = b.abs() * torch.exp2(-e.float()).unsqueeze(-1)
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).byte()
    code = (code | (torch.signbit(b).byte() << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).byte()


def _decode(codes, exps):
    """The f32 values of MXFP4 codes and exponents."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    x = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)
    return (x.unflatten(-1, (-1, 32)) * torch.exp2(exps.float() - 127).unsqueeze(-1)).flatten(-2)


def _f16(x):
    """The cache's f16: nearest even, magnitudes below the normal range to zero."""
    return torch.where(x.abs() < 2.0 ** -14, x * 0, x).half()


def _batch(c, g):
    s = _State()
    s.c, s.g = c, g
    seqs = _seqs(c)
    s.lens = [n for n, _ in seqs]
    s.len = torch.tensor(s.lens, dtype=torch.int32, device="cuda")
    ends = [0]
    for _, r in seqs:
        ends.append(ends[-1] + r)
    s.n_rows, s.max_rows = ends[-1], max(r for _, r in seqs)
    s.row0 = torch.tensor(ends, dtype=torch.int32, device="cuda")
    s.max_pages = max(-(-n // c["page"]) for n in s.lens)
    # pages handed out in random order; entries behind a sequence's last page are never read
    need = [-(-n // c["page"]) for n in s.lens]
    s.n_pages = sum(need) + 1
    order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
    at = torch.arange(s.max_pages, device="cuda")[None] + torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")[:, None]
    s.pages = torch.where(torch.arange(s.max_pages, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None],
                          order[at.clamp(max=s.n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32)).int().contiguous()
    shape = (s.n_pages, c["nkv"], c["page"], c["hd"])
    s.ks = s.vs = None
    if c["kind"] == "append":       # what it held before does not matter: only the new rows are looked at
        if c["dt"] == "f16":
            s.k, s.v = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        else:
            s.k, s.v = (torch.zeros(shape[:3] + (c["hd"] // 2,), dtype=torch.uint8, device="cuda") for _ in range(2))
            s.ks, s.vs = (torch.full(shape[:3] + (c["hd"] // 32,), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    elif c["dt"] == "f16":
        s.k, s.v = _normal(shape, g).half(), _normal(shape, g).half()
    else:
        s.k, s.ks = _encode(_normal(shape, g))
        s.v, s.vs = _encode(_normal(shape, g))
    return s


def _own_batch(s):
    from midge_amd import kv
    c, p = s.c, lambda t: t.data_ptr() if t is not None else 0
    s.cache = kv.KVCache(F16 if c["dt"] == "f16" else MXFP4, c["nkv"], c["hd"], c["page"], s.n_pages, p(s.k), p(s.v), p(s.ks), p(s.vs))
    one = s.max_rows == 1
    s.batch = kv.KVBatch(c["seqs"], s.n_rows, s.max_rows, s.max_pages, 0 if one else p(s.row0), p(s.len), p(s.pages))


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "logprobs":
        s = _State()
        s.c = case
        n, v = case["n"], case["vocab"]
        s.logits = _normal((n, v), g, case["spread"])
        s.ids = torch.randint(0, v, (n, case["ids"]), device="cuda", generator=g, dtype=torch.int32)
        # a sampled token is a likely one
        if case["ids"]:
            s.ids[:, 0] = (s.logits + _normal((n, v), g, 1.0)).argmax(-1).int()
        s.top = min(case["top"], v)
        s.lp = torch.empty((n, case["ids"]), device="cuda")
        s.entropy = torch.empty(n, device="cuda")
        s.top_id = torch.empty((n, s.top), dtype=torch.int32, device="cuda")
        s.top_lp = torch.empty((n, s.top), device="cuda")
        if own:
            import midge_amd
            from midge_amd import moe
            midge_amd.init(0)
            s.ws_bytes = moe.logprobs_ws(n, v, s.top)
            s.ws = torch.zeros(s.ws_bytes, dtype=torch.uint8, device="cuda")
    else:
        s = _batch(case, g)
        nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
        if case["kind"] == "append":
            # the rows of one fused projection
            s.qkv = _normal((s.n_rows, (nh + 2 * nkv) * hd), g)
            s.bq, s.bk, s.bv = (_normal(n * hd, g, 0.2) for n in (nh, nkv, nkv))
            s.qn, s.kn = (_normal(hd, g, 0.1, 1.0) for _ in range(2)) if case["norm"] else (None, None)
            ang = torch.arange(max(s.lens), device="cuda").double()[:, None] * 150000.0 ** (-torch.arange(hd // 2, device="cuda").double() / (hd // 2))
            s.cos, s.sin = ang.cos().float(), ang.sin().float()
            s.q_out = torch.empty((s.n_rows, nh * hd), device="cuda")
            s.k_out, s.v_out = (torch.empty((s.n_rows, nkv * hd), device="cuda") for _ in range(2))
        else:
            s.q = _normal((s.n_rows, nh * hd), g, 1.5)
            s.sink = _normal(nh, g) if case["sink"] else None
            s.out = torch.empty((s.n_rows, nh * hd), device="cuda")
        if own:
            import midge_amd
            from midge_amd import kv
            midge_amd.init(0)
            _own_batch(s)
            if case["kind"] == "append":
                w = (nh + 2 * nkv) * hd
                p, at = lambda t: t.data_ptr() if t is not None else 0, s.qkv.data_ptr()
                s.rows = kv.KVRows(nh, s.cos.shape[0], EPS, at, at + 4 * nh * hd, at + 4 * (nh + nkv) * hd, w, w, w, p(s.q_out),
                                   p(s.bq), p(s.bk), p(s.bv), p(s.qn), p(s.kn), p(s.cos), p(s.sin))
            else:
                s.ws_bytes = kv.attention_ws(s.cache, s.batch, nh)
                s.ws = torch.zeros(max(s.ws_bytes, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms

def _where(s):
    """Of each row: its sequence, its place in it, its position."""
    r = torch.arange(s.n_rows, device="cuda")
    q = torch.searchsorted(s.row0[1:].contiguous(), r, right=True)
    i = r - s.row0[q]
    return q, i, s.len[q] - (s.row0[q + 1] - s.row0[q]) + i


def _prepared_rows(s, x, bias, norm, pos):
    """x[n][heads][hd] with bias, norm and rotation, in 64 bits, rounded once to f32."""
    x = x.double() + bias.double().view(x.shape[1:])
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.double()
    if pos is not None:
        a, b = x.chunk(2, -1)
        c, n = s.cos[pos].double()[:, None], s.sin[pos].double()[:, None]
        x = torch.cat((a * c - b * n, b * c + a * n), -1)
    return x.float()


def _append_plain(s):
    c = s.c
    q, k, v = s.qkv.unflatten(-1, (-1, c["hd"])).split((c["nh"], c["nkv"], c["nkv"]), 1)
    seq, _, pos = _where(s)
    page, slot = s.pages[seq, pos // c["page"]].long(), pos % c["page"]
    k = _prepared_rows(s, k, s.bk, s.kn, pos)
    v = _prepared_rows(s, v, s.bv, None, None)
    if c["dt"] == "f16":
        s.k[page, :, slot], s.v[page, :, slot] = _f16(k), _f16(v)
        k, v = s.k[page, :, slot].float(), s.v[page, :, slot].float()
    else:
        (s.k[page, :, slot], s.ks[page, :, slot]), (s.v[page, :, slot], s.vs[page, :, slot]) = _encode(k), _encode(v)
        k, v = _decode(s.k[page, :, slot], s.ks[page, :, slot]), _decode(s.v[page, :, slot], s.vs[page, :, slot])
    return {"q": _prepared_rows(s, q, s.bq, s.qn, pos).flatten(1), "k": k.flatten(1), "v": v.flatten(1)}


def _gathered(s, x, xs):
    """A batch's pages in order, as f32 [seqs][nkv][max_pages * page][hd]."""
    at = s.pages.clamp(min=0).long()
    x = x[at].float() if xs is None else _decode(x[at], xs[at])
    return x.transpose(1, 2).flatten(2, 3)


def _attention_plain(s):
    c = s.c
    n, nkv, hd, group = c["seqs"], c["nkv"], c["hd"], c["nh"] // c["nkv"]
    k, v = _gathered(s, s.k, s.ks), _gathered(s, s.v, s.vs)
    i = torch.arange(s.max_rows, device="cuda")[None]
    rows = s.row0[1:] - s.row0[:-1]
    q = s.q[(s.row0[:-1, None] + i).clamp(max=s.n_rows - 1)]                     # [seqs][max_rows][nh * hd]
    q = q.view(n, s.max_rows, nkv, group, hd).transpose(1, 2).reshape(n, nkv, -1, hd)
    a = q @ k.transpose(2, 3).contiguous() * hd ** -0.5
    pos = (s.len - rows)[:, None] + i                                             # [seqs][max_rows]
    t = torch.arange(k.shape[2], device="cuda")
    hide = t > pos[..., None]
    if c["window"]:
        hide = hide | (t <= pos[..., None] - c["window"])
    a = a.view(n, nkv, s.max_rows, group, -1).masked_fill_(hide[:, None, :, None], -math.inf)
    m = a.amax(-1, keepdim=True)
    if s.sink is not None:
        m = torch.maximum(m, s.sink.view(1, nkv, 1, group, 1))
    e = a.sub_(m).exp_()
    den = e.sum(-1, keepdim=True)
    if s.sink is not None:
        den = den + (s.sink.view(1, nkv, 1, group, 1) - m).exp()
    o = (e.view(n, nkv, -1, e.shape[-1]) @ v).view(n, nkv, s.max_rows, group, hd) / den
    seq, i, _ = _where(s)
    return o.transpose(1, 2).flatten(2)[seq, i]


def _logprobs_plain(s):
    x = s.logits
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    z = e.sum(-1, keepdim=True)
    entropy = (z.log() - (e * d).sum(-1, keepdim=True) / z)[:, 0]
    top, at = torch.sort(x, dim=-1, descending=True, stable=True) if s.top else (x[:, :0], torch.zeros_like(x[:, :0], dtype=torch.int64))
    return {"lp": (x.gather(1, s.ids.long()) - m) - z.log(), "entropy": entropy, "top_id": at[:, :s.top].int(),
            "top_lp": (top[:, :s.top] - m) - z.log()}


# -------------------------------------------------------------------- run

def _run_own(s):
    from midge_amd import kv, moe
    c = s.c
    if c["kind"] == "logprobs":
        p = lambda t: t.data_ptr() if t.numel() else 0     # noqa: E731
        moe.logprobs_dev(s.logits.data_ptr(), c["vocab"], c["n"], c["vocab"], p(s.ids), c["ids"], s.top, p(s.lp), s.entropy.data_ptr(),
                         p(s.top_id), p(s.top_lp), s.ws.data_ptr(), s.ws_bytes)
        return {"lp": s.lp, "entropy": s.entropy, "top_id": s.top_id, "top_lp": s.top_lp}
    if c["kind"] == "append":
        kv.append_dev(s.cache, s.batch, s.rows)
        kv.read_dev(s.cache, s.batch, s.k_out.data_ptr(), s.v_out.data_ptr())
        return {"q": s.q_out, "k": s.k_out, "v": s.v_out}
    kv.attention_dev(s.cache, s.batch, c["nh"], s.q.data_ptr(), s.out.data_ptr(), s.ws.data_ptr(), s.ws_bytes, c["hd"] ** -0.5, c["window"],
                     s.sink.data_ptr() if s.sink is not None else 0)
    return s.out


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}[state.c["kind"]](state)


# ------------------------------------------------------------------ exact

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _stored(x, dt):
    """What a cache of type dt holds of f32 values x[..., hd], in 64 bits."""
    x = x.double()
    if dt == "f16":
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14))) - 10)
        return torch.where(x.abs() < 2.0 ** -14, 0.0, torch.round(x / step) * step)     # round() goes to even
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -13)
    for e in range(-12, 14):
        scale = torch.where(top > 7 * scale, 2.0 ** e, scale)
    levels = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    # the nearest level; of two equally near ones that of the even code
    far = (b.abs() / scale)[..., None] - levels
    code = (far.abs() + 1e-9 * (torch.arange(8, device="cuda") % 2)).argmin(-1)
    return (torch.sign(b) * levels[code] * scale).flatten(-2)


def _exact_append(s):
    c, hd = s.c, s.c["hd"]
    pos = torch.cat([torch.arange(n - r, n) for n, r in _seqs(c)]).cuda()

    def rows(at, heads, bias, norm, turn):
        x = s.qkv[:, at * hd:(at + heads) * hd].double() + bias.double()
        x = x.view(-1, heads, hd)
        if norm is not None:
            x = x * (x.square().sum(-1, keepdim=True) / hd + EPS).rsqrt() * norm.double()
        if turn:
            z = torch.complex(x[..., :hd // 2], x[..., hd // 2:])
            z = z * torch.complex(s.cos[pos].double(), s.sin[pos].double())[:, None]
            x = torch.cat((z.real, z.imag), -1)
        return x
    q = rows(0, c["nh"], s.bq, s.qn, True)
    k = rows(c["nh"], c["nkv"], s.bk, s.kn, True).float()
    v = rows(c["nh"] + c["nkv"], c["nkv"], s.bv, None, False).float()
    return {"q": q.flatten(1), "k": _stored(k, c["dt"]).flatten(1), "v": _stored(v, c["dt"]).flatten(1)}


def _exact_attention(s):
    c, out, r0 = s.c, [], 0
    nkv, hd, group = c["nkv"], c["hd"], c["nh"] // c["nkv"]
    levels = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device="cuda")

    def tokens(x, xs, pages, n):
        x = x[pages]
        if xs is None:
            x = x.double()
        else:
            lo, hi = levels[(x % 16).long()], levels[(x // 16).long()]
            x = torch.stack((lo, hi), -1).flatten(-2) * torch.exp2(xs[pages].double() - 127).repeat_interleave(32, -1)
        return x.transpose(0, 1).reshape(nkv, -1, hd)[:, :n]
    for b, (n, r) in enumerate(_seqs(c)):
        pages = s.pages[b, :-(-n // c["page"])].long()
        k, v = tokens(s.k, s.ks, pages, n), tokens(s.v, s.vs, pages, n)
        q = s.q[r0:r0 + r].double().view(r, nkv, group, hd)
        for i in range(0, r, 500):          # some rows at a time: the scores fit
            j = min(i + 500, r)
            a = torch.matmul(q[i:j].permute(1, 2, 0, 3).reshape(nkv, -1, hd), k.transpose(1, 2).contiguous()) / math.sqrt(hd)
            a = a.view(nkv, group, j - i, n)
            at, t = torch.arange(n - r + i, n - r + j, device="cuda")[:, None], torch.arange(n, device="cuda")
            seen = (t <= at) & (t > at - (c["window"] or n))
            a = torch.where(seen, a, -math.inf)
            if s.sink is not None:
                a = torch.cat((a, s.sink.double().view(nkv, group, 1, 1).expand(-1, -1, j - i, 1)), -1)
            p = torch.softmax(a, -1)[..., :n].reshape(nkv, -1, n)
            out.append(torch.matmul(p, v).view(nkv, group, j - i, hd).permute(2, 0, 1, 3).reshape(j - i, -1))
        r0 += r
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attention":
        return _exact_attention(s)
    lp, ent, ids, tops = [], [], [], []
    for x, want in zip(s.logits, s.ids):
        p = torch.log_softmax(x.double(), -1)
        lp.append(p[want.long()])
        ent.append(-(p.exp() * p).sum())
        order = torch.argsort(x, descending=True, stable=True)[:s.top]
        ids.append(order.int())
        tops.append(p[order])
    return {"lp": torch.stack(lp), "entropy": torch.stack(ent), "top_id": torch.stack(ids), "top_lp": torch.stack(tops)}


# ------------------------------------------------------------------- work

def work(case):
    c = case
    if c["kind"] == "logprobs":
        return {"bytes": c["n"] * (4 * c["vocab"] + 8 * c["ids"] + 4 + 8 * c["top"]), "flops": 6 * c["n"] * c["vocab"]}
    hd, seqs = c["hd"], _seqs(c)
    token = c["nkv"] * (4 * hd if c["dt"] == "f16" else hd + hd // 16)      # k and v of one token
    rows = sum(r for _, r in seqs)
    if c["kind"] == "append":
        return {"bytes": rows * (4 * hd * (2 * c["nh"] + 2 * c["nkv"]) + 2 * token + 8 * hd * c["nkv"]), "flops": 10 * rows * hd * (c["nh"] + 2 * c["nkv"])}
    seen = pairs = 0
    for n, r in seqs:
        w = c["window"] or n
        seen += min(n, w + r - 1)
        pairs += sum(min(p + 1, w) for p in range(n - r, n))
    return {"bytes": seen * token + 8 * rows * c["nh"] * hd, "flops": 4 * hd * c["nh"] * pairs}
