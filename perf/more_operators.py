"""The operators of speculative decoding whose speed is kept in view: several
tokens of a sequence, drafted as a tree, go through the model in one step.

    append     the rows of a batch of trees: as a batch's new rows, but a row's
               slot is its place in the tree's order and its position its depth
               (mh_kv_tree_append_dev), and the stored values read back
    attention  each row over its sequence's cached tokens and its own ancestors
               (mh_kv_tree_attention_dev)
    verify     which drafts the target's probabilities keep, from given random
               numbers, and the token after them (mh_verify_dev)
    keep       the kept rows' k and v of all layers moved to the slots behind
               the cached tokens (mh_kv_keep_dev)

Head layouts are those of the models the framework serves (64 query heads on
8 of 64; 32 on 8 and 32 on 4 of 128) and generic ones. k and v are normal
values through the cache's own encoding, pages lie in random order.
"""
import math

import torch

own = False

EPS = 1e-5
F16, MXFP4 = 0, 1       # cache types, as MH_KV_F16 and MH_KV_MXFP4
MOST = 64               # rows of a tree


# ------------------------------------------------------------------ cases

def _heads(nh, nkv, hd):
    return dict(nh=nh, nkv=nkv, hd=hd)


_A, _B, _C = _heads(64, 8, 64), _heads(32, 8, 128), _heads(32, 4, 128)


def _kv(kind, heads, dt, seqs, rows, lo, hi, page=64, name=None, **more):
    """`seqs` sequences of lo..hi tokens (evenly spread over the logarithm), the last of each, `rows` or somewhat fewer, a tree."""
    c = dict(kind=kind, dt=dt, seqs=seqs, rows=rows, lo=lo, hi=hi, page=page, **heads)
    c.update({"attention": dict(window=0, sink=False), "append": dict(norm=False), "keep": dict(layers=1)}[kind])
    c.update(more)
    return dict(c, name=name) if name else c


def _verify(seqs, rows, vocab, q=False, chain=False, temp=0.75, name=None):
    c = dict(kind="verify", seqs=seqs, rows=rows, vocab=vocab, q=q, chain=chain, temp=temp)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the draft tree of one chat
        _kv("append", _A, "mxfp4", 1, 16, 1044, 1044, name="append_b1"),
        # a serving batch's trees, with norms of q and k
        _kv("append", _C, "f16", 64, 8, 17, 9000, norm=True, page=16, name="append_b64"),
        # one chat: a short tree and a wide one, at a usual and at a very long context
        _kv("attention", _A, "mxfp4", 1, 8, 4100, 4100, sink=True, name="tree_b1_4k"),
        _kv("attention", _A, "mxfp4", 1, 64, 131071, 131071, sink=True, name="tree_b1_128k"),
        # a serving batch with contexts of all lengths
        _kv("attention", _A, "mxfp4", 32, 13, 100, 16000, sink=True, name="tree_b32"),
        # the same from an f16 cache, wider heads
        _kv("attention", _B, "f16", 16, 25, 500, 8191, page=16, name="tree_b16_f16"),
        # a sliding layer of a serving batch
        _kv("attention", _A, "mxfp4", 32, 13, 100, 16000, window=128, sink=True, name="tree_b32_window"),
        # a chat's tree; a serving batch's trees; drafts that were drawn from a small model's probabilities
        _verify(1, 8, 201088, name="verify_b1"),
        _verify(32, 8, 201088, name="verify_b32"),
        _verify(16, 6, 201088, q=True, chain=True, name="verify_b16_q"),
        # all layers' caches of a chat and of a serving batch
        _kv("keep", _A, "f16", 1, 16, 4100, 4100, layers=36, name="keep_b1"),
        _kv("keep", _C, "f16", 64, 13, 40, 900, page=16, layers=24, name="keep_b64"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LAYOUTS = [_A, _A, _B, _C, _heads(16, 16, 64), _heads(24, 2, 96), _heads(8, 1, 256), _heads(40, 10, 32), _heads(12, 4, 192)]


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "verify", "verify", "keep"])
    if kind == "verify":
        vocab, rows = _log(rng, 1000, 201088), _log(rng, 1, MOST)
        q = rng.choice([False, True])
        seqs = _log(rng, 1, max(1, min(64, (25 if q else 50) * 10 ** 6 // vocab // rows)))
        return _verify(seqs, rows, vocab, q, rng.choice([False, False, True]), rng.choice([0.0, 0.3, 0.75, 1.0, 1.0, 1.5]))
    heads, dt, page = rng.choice(_LAYOUTS), rng.choice(["mxfp4", "mxfp4", "f16"]), rng.choice([16, 32, 64, 128, 256])
    seqs, rows = _log(rng, 1, 64), _log(rng, 1, MOST)
    if kind == "append":
        lo = rows + _log(rng, 1, 2000)
        return _kv(kind, heads, dt, seqs, rows, lo, lo + rng.choice([0, _log(rng, 1, 4000)]), page, norm=rng.choice([False, True]))
    if kind == "keep":
        lo = rows + _log(rng, 1, 600)
        return _kv(kind, heads, dt, seqs, rows, lo, lo + rng.choice([0, 50]), page, layers=rng.choice([1, 8, 24]) if dt == "f16" else rng.randint(1, 3))
    lo = rows + _log(rng, 1, 400000 // seqs // heads["nkv"])
    lo = min(lo, rows + 200 * 10 ** 6 // (seqs * rows * heads["nh"]))
    return _kv(kind, heads, dt, seqs, rows, lo, lo + rng.choice([0, lo]), page, window=rng.choice([0, 0, 128, 1000, 3]), sink=rng.choice([False, True]))


def _seqs(c):
    """[(tokens, tree rows)] of a batch; the trees differ in size a little."""
    n, out = c["seqs"], []
    for i in range(n):
        length = int(round(c["lo"] * (c["hi"] / c["lo"]) ** (i / (n - 1)))) if n > 1 else c["lo"]
        out.append((length, max(1, c["rows"] - i * 5 % max(1, c["rows"] // 2))))
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


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


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


def _trees(s, rows, g, chain=False):
    """row0 and, of each row, its parent's place in the tree: -1 for the first, any earlier row for the others, later ones likelier."""
    ends = [0]
    for r in rows:
        ends.append(ends[-1] + r)
    s.n_rows, s.max_rows, s.row0 = ends[-1], max(rows), _ints(ends)
    s.seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), _ints(rows).long())
    s.at = torch.arange(s.n_rows, device="cuda") - s.row0[s.seq]
    u = torch.rand(s.n_rows, device="cuda", generator=g)
    up = s.at - 1 if chain else (s.at * u.sqrt()).long().clamp(max=s.at - 1)
    s.parent = torch.where(s.at > 0, up, torch.full_like(up, -1)).int()


def _batch(c, g):
    s = _State()
    s.c = c
    seqs = _seqs(c)
    s.lens = [n for n, _ in seqs]
    s.len = _ints(s.lens)
    _trees(s, [r for _, r in seqs], g)
    need = [-(-n // c["page"]) for n in s.lens]
    s.max_pages = max(need)
    # pages handed out in random order; entries behind a sequence's last page are never read
    s.n_pages = sum(need) + 1
    order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
    at = torch.arange(s.max_pages, device="cuda")[None] + torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")[:, None]
    s.pages = torch.where(torch.arange(s.max_pages, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None],
                          order[at.clamp(max=s.n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32)).int().contiguous()
    shape = (c.get("layers", 1), s.n_pages, c["nkv"], c["page"], c["hd"])
    s.ks = s.vs = None
    if c["kind"] == "append":       # what it held before does not matter: only the new rows are looked at
        if c["dt"] == "f16":
            s.k, s.v = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        else:
            s.k, s.v = (torch.zeros(shape[:4] + (c["hd"] // 2,), dtype=torch.uint8, device="cuda") for _ in range(2))
            s.ks, s.vs = (torch.full(shape[:4] + (c["hd"] // 32,), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    elif c["dt"] == "f16":
        s.k, s.v = _normal(shape, g).half(), _normal(shape, g).half()
    else:
        s.k, s.ks = _encode(_normal(shape, g))
        s.v, s.vs = _encode(_normal(shape, g))
    return s


def _own_batch(s):
    from midge_amd import kv
    c, p = s.c, lambda t, i: t[i].data_ptr() if t is not None else 0
    s.caches = [kv.KVCache(F16 if c["dt"] == "f16" else MXFP4, c["nkv"], c["hd"], c["page"], s.n_pages, p(s.k, i), p(s.v, i), p(s.ks, i), p(s.vs, i))
                for i in range(s.k.shape[0])]
    s.batch = kv.KVBatch(c["seqs"], s.n_rows, s.max_rows, s.max_pages, s.row0.data_ptr(), s.len.data_ptr(), s.pages.data_ptr())


def _drafts(case, g):
    """Logits with a few likely tokens a row over a broad rest; drafts as a smaller model makes them, whose logits are off by some noise:
    its likeliest tokens, or tokens drawn from its probabilities q."""
    s = _State()
    s.c, v = case, case["vocab"]
    rows = [max(1, case["rows"] - i * 5 % max(1, case["rows"] // 2)) for i in range(case["seqs"])]
    _trees(s, rows, g, case["chain"])
    n = s.n_rows
    s.logits = _normal((n, v), g, 2.0)
    likely = torch.randint(0, v, (n, 16), device="cuda", generator=g)
    s.logits.scatter_(1, likely, _normal((n, 16), g, 2.0, 2.0 + math.log(v)))
    up = (s.row0[s.seq] + s.parent.clamp(min=0)).long()       # the row whose distribution a draft comes from
    off = _normal((n, 16), g, 1.0)
    s.q = None
    if case["q"]:
        s.q = torch.softmax((s.logits.scatter_add(1, likely, off)) / (case["temp"] or 1.0), -1)
        # drawn by the smallest of exponential variates over the probabilities; all at once where they fit
        s.token = torch.cat([(torch.empty((len(r), v), device="cuda").exponential_(generator=g) / s.q[r]).argmin(-1) for r in up.split(256)]).int()
    else:
        best = s.logits.gather(1, likely)[up] + _normal((n, 16), g, 2.0)
        s.token = likely[up].gather(1, best.argmax(-1, keepdim=True))[:, 0].int()
    s.u = torch.rand(n, device="cuda", generator=g)
    return s


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "verify":
        s = _drafts(case, g)
        if own:
            import midge_amd
            from midge_amd import moe
            midge_amd.init(0)
            seqs, p = case["seqs"], lambda t: t.data_ptr() if t is not None else 0
            s.n_kept, s.next = torch.empty(seqs, dtype=torch.int32, device="cuda"), torch.empty(seqs, dtype=torch.int32, device="cuda")
            s.kept = torch.empty((seqs, s.max_rows), dtype=torch.int32, device="cuda")
            s.draft = moe.Draft(seqs, s.n_rows, s.max_rows, p(s.row0), 0 if case["chain"] else p(s.parent), p(s.token), p(s.u), case["vocab"],
                                p(s.logits), case["vocab"], case["temp"], p(s.q), case["vocab"])
            s.ws_bytes = moe.verify_ws(seqs, s.n_rows, case["vocab"])
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
        elif case["kind"] == "attention":
            s.q = _normal((s.n_rows, nh * hd), g, 1.5)
            s.sink = _normal(nh, g) if case["sink"] else None
            s.out = torch.empty((s.n_rows, nh * hd), device="cuda")
        else:
            # a path from the root of each tree, of any length: what a verification keeps
            depth = torch.rand(case["seqs"], s.max_rows, device="cuda", generator=g) < 0.7
            kept = torch.full((case["seqs"], s.max_rows), -1, dtype=torch.int32)
            parents, row0, far = s.parent.tolist(), s.row0.tolist(), depth.tolist()
            n_kept = []
            for i in range(case["seqs"]):
                path, cur = [0], 0
                for r in range(1, row0[i + 1] - row0[i]):
                    if parents[row0[i] + r] == cur and far[i][r]:
                        path.append(r)
                        cur = r
                kept[i, :len(path)] = torch.tensor(path, dtype=torch.int32)
                n_kept.append(len(path))
            s.kept, s.n_kept, s.len_out = kept.cuda(), _ints(n_kept), torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
            if case["dt"] != "f16":     # the rows' slots afterwards, read back
                s.back = torch.empty((case["layers"], 2, s.n_rows, nkv * hd), device="cuda")
        if own:
            import midge_amd
            from midge_amd import kv
            midge_amd.init(0)
            _own_batch(s)
            p = lambda t: t.data_ptr() if t is not None else 0      # noqa: E731
            if case["kind"] == "append":
                w, at = (nh + 2 * nkv) * hd, s.qkv.data_ptr()
                s.rows = kv.KVRows(nh, s.cos.shape[0], EPS, at, at + 4 * nh * hd, at + 4 * (nh + nkv) * hd, w, w, w, p(s.q_out),
                                   p(s.bq), p(s.bk), p(s.bv), p(s.qn), p(s.kn), p(s.cos), p(s.sin))
            elif case["kind"] == "attention":
                s.ws_bytes = kv.tree_attention_ws(s.caches[0], s.batch, nh)
                s.ws = torch.zeros(max(s.ws_bytes, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms

def _ancestors(s):
    """[seqs][max_rows][max_rows]: row i of a tree sees row j: j is i or an ancestor of it."""
    n = s.max_rows
    one = torch.zeros((s.row0.numel() - 1, n, n), device="cuda")
    i = s.at > 0
    one[s.seq[i], s.at[i], s.parent[i].long()] = 1.0
    see = one + torch.eye(n, device="cuda")
    for _ in range(6):      # (paths of up to 2^6 steps)
        see = (see @ see).clamp(max=1.0)
    return see > 0.5


def _depths(s):
    return _ancestors(s).sum(-1) - 1


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


def _base(s):
    """Of each sequence: its tokens before the tree."""
    return (s.len - (s.row0[1:] - s.row0[:-1])).long()


def _append_plain(s):
    c = s.c
    q, k, v = s.qkv.unflatten(-1, (-1, c["hd"])).split((c["nh"], c["nkv"], c["nkv"]), 1)
    base = _base(s)[s.seq]
    pos, t = base + _depths(s)[s.seq, s.at], base + s.at
    page, slot = s.pages[s.seq, t // c["page"]].long(), t % c["page"]
    k = _prepared_rows(s, k, s.bk, s.kn, pos)
    v = _prepared_rows(s, v, s.bv, None, None)
    if c["dt"] == "f16":
        s.k[0][page, :, slot], s.v[0][page, :, slot] = _f16(k), _f16(v)
        k, v = s.k[0][page, :, slot].float(), s.v[0][page, :, slot].float()
    else:
        (s.k[0][page, :, slot], s.ks[0][page, :, slot]), (s.v[0][page, :, slot], s.vs[0][page, :, slot]) = _encode(k), _encode(v)
        k, v = _decode(s.k[0][page, :, slot], s.ks[0][page, :, slot]), _decode(s.v[0][page, :, slot], s.vs[0][page, :, slot])
    return {"q": _prepared_rows(s, q, s.bq, s.qn, pos).flatten(1), "k": k.flatten(1), "v": v.flatten(1)}


def _gathered(s, x, xs):
    """A batch's pages in order, as f32 [seqs][nkv][max_pages * page][hd]."""
    at = s.pages.clamp(min=0).long()
    x = x[0][at].float() if xs is None else _decode(x[0][at], xs[0][at])
    return x.transpose(1, 2).flatten(2, 3)


def _attention_plain(s):
    c = s.c
    n, nkv, hd, group = c["seqs"], c["nkv"], c["hd"], c["nh"] // c["nkv"]
    k, v = _gathered(s, s.k, s.ks), _gathered(s, s.v, s.vs)
    i = torch.arange(s.max_rows, device="cuda")[None]
    q = s.q[(s.row0[:-1, None] + i).clamp(max=s.n_rows - 1)]                     # [seqs][max_rows][nh * hd]
    q = q.view(n, s.max_rows, nkv, group, hd).transpose(1, 2).reshape(n, nkv, -1, hd)
    a = q @ k.transpose(2, 3).contiguous() * hd ** -0.5
    see, base = _ancestors(s), _base(s)
    depth = see.sum(-1) - 1
    t = torch.arange(k.shape[2], device="cuda")[None]
    own_row = t - base[:, None]                                                   # a token's row of the tree
    in_tree = (own_row >= 0) & (own_row < s.max_rows)
    at = own_row.clamp(0, s.max_rows - 1)
    hide = (own_row >= 0)[:, None] & ~(see.gather(2, at[:, None].expand(-1, s.max_rows, -1)) & in_tree[:, None])
    if c["window"]:
        where = torch.where(own_row >= 0, base[:, None] + depth.gather(1, at), t)     # a token's position
        hide = hide | (where[:, None] <= (base[:, None] + depth)[..., None] - c["window"])
    a = a.view(n, nkv, s.max_rows, group, -1).masked_fill_(hide[:, None, :, None], -math.inf)
    m = a.amax(-1, keepdim=True)
    if s.sink is not None:
        m = torch.maximum(m, s.sink.view(1, nkv, 1, group, 1))
    e = a.sub_(m).exp_()
    den = e.sum(-1, keepdim=True)
    if s.sink is not None:
        den = den + (s.sink.view(1, nkv, 1, group, 1) - m).exp()
    o = (e.view(n, nkv, -1, e.shape[-1]) @ v).view(n, nkv, s.max_rows, group, hd) / den
    return o.transpose(1, 2).flatten(2)[s.seq, s.at]


def _verify_plain(s):
    """All sequences together, row by row of the trees in order; in 64 bits."""
    c, row0 = s.c, s.row0[:-1].long()
    seqs, n = c["seqs"], s.max_rows
    rows = (s.row0[1:] - s.row0[:-1]).long()
    x = s.logits
    m, first = x.max(-1, keepdim=True)[0], x.argmax(-1)
    if c["temp"] > 0:
        heat = torch.tensor(c["temp"], dtype=torch.float32).double().item()
        e = ((x.double() - m.double()) / heat).exp()
        p = e / e.sum(-1, keepdim=True)
    else:
        p = torch.zeros_like(x, dtype=torch.float64).scatter_(1, first[:, None], 1.0)
    one = torch.arange(seqs, device="cuda")
    cur = torch.zeros(seqs, dtype=torch.int64, device="cuda")
    kept = torch.full((seqs, n), -1, dtype=torch.int32, device="cuda")
    kept[:, 0] = 0
    n_kept = torch.ones(seqs, dtype=torch.int64, device="cuda")
    left = p[row0]                              # what is left of the current row's probabilities, and its sum
    alpha, w = torch.zeros(seqs, dtype=torch.float64, device="cuda"), torch.ones(seqs, dtype=torch.float64, device="cuda")
    drawn = s.q is not None and c["temp"] > 0
    for i in range(1, n):
        r = (row0 + i).clamp(max=s.n_rows - 1)
        child = (i < rows) & (s.parent[r] == cur)
        t, u = s.token[r].long(), s.u[r].double()
        qc = s.q[row0 + cur, t].double() if drawn else 1.0
        yes = child & (u * qc * w < left[one, t])
        no = child & ~yes
        if drawn:
            alpha = torch.where(no, alpha + w, alpha)
            rest = (p[row0 + cur] - alpha[:, None] * s.q[row0 + cur].double()).clamp(min=0)
        else:
            rest = left.scatter(1, t[:, None], 0.0)
        left = torch.where(no[:, None], rest, left)
        w = torch.where(no, left.sum(-1), w)
        kept[one, torch.where(yes, n_kept, n - 1)] = torch.where(yes, i, kept[:, n - 1]).int()
        n_kept = n_kept + yes
        cur = torch.where(yes, i, cur)
        left = torch.where(yes[:, None], p[row0 + cur], left)
        alpha, w = torch.where(yes, 0.0, alpha), torch.where(yes, 1.0, w)
    left = torch.where((left.sum(-1) > 0)[:, None], left, p[row0 + cur])
    run = left.cumsum(-1)
    after = torch.searchsorted(run, s.u[row0].double()[:, None] * run[:, -1:], right=True)[:, 0].clamp(max=c["vocab"] - 1)
    return {"n_kept": n_kept.int(), "kept": kept, "next": after.int()}


def _keep_plain(s):
    c = s.c
    j = torch.arange(s.max_rows, device="cuda")[None]
    seq, at = torch.nonzero(j < s.n_kept[:, None], as_tuple=True)
    base = _base(s)
    old, new = base[seq] + s.kept[seq, at], base[seq] + at
    page = c["page"]
    for x in (s.k, s.v, s.ks, s.vs):
        if x is not None:
            x[:, s.pages[seq, new // page].long(), :, new % page] = x[:, s.pages[seq, old // page].long(), :, old % page]
    length = (base + s.n_kept).int()
    if c["dt"] == "f16":
        return {"k": s.k, "v": s.v, "len": length}
    t = base[s.seq] + s.at
    at = s.pages[s.seq, t // page].long(), slice(None), t % page
    back = [torch.stack([_decode(x[i][at], xs[i][at]).flatten(1) for x, xs in ((s.k, s.ks), (s.v, s.vs))]) for i in range(c["layers"])]
    return {"kv": torch.stack(back), "len": length}


# -------------------------------------------------------------------- run

def _run_own(s):
    from midge_amd import kv, moe
    c = s.c
    if c["kind"] == "verify":
        moe.verify_dev(s.draft, s.n_kept.data_ptr(), s.kept.data_ptr(), s.next.data_ptr(), s.ws.data_ptr(), s.ws_bytes)
        return {"n_kept": s.n_kept, "kept": s.kept, "next": s.next}
    if c["kind"] == "append":
        kv.tree_append_dev(s.caches[0], s.batch, s.parent.data_ptr(), s.rows)
        kv.read_dev(s.caches[0], s.batch, s.k_out.data_ptr(), s.v_out.data_ptr())
        return {"q": s.q_out, "k": s.k_out, "v": s.v_out}
    if c["kind"] == "attention":
        kv.tree_attention_dev(s.caches[0], s.batch, s.parent.data_ptr(), c["nh"], s.q.data_ptr(), s.out.data_ptr(), s.ws.data_ptr(), s.ws_bytes,
                              c["hd"] ** -0.5, c["window"], s.sink.data_ptr() if s.sink is not None else 0)
        return s.out
    kv.keep_dev(s.caches, s.batch, s.n_kept.data_ptr(), s.kept.data_ptr(), s.len_out.data_ptr())
    if c["dt"] == "f16":
        return {"k": s.k, "v": s.v, "len": s.len_out}
    for cache, (k, v) in zip(s.caches, s.back):
        kv.read_dev(cache, s.batch, k.data_ptr(), v.data_ptr())
    return {"kv": s.back, "len": s.len_out}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append_plain, "attention": _attention_plain, "verify": _verify_plain, "keep": _keep_plain}[state.c["kind"]](state)


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


def _paths(s):
    """Of each sequence, of each of its rows: the rows from the root to it."""
    up, ends, out = s.parent.tolist(), s.row0.tolist(), []
    for a, b in zip(ends, ends[1:]):
        paths = []
        for i in range(b - a):
            paths.append((paths[up[a + i]] if up[a + i] >= 0 else []) + [i])
        out.append(paths)
    return out


def _exact_append(s):
    c, hd = s.c, s.c["hd"]
    pos = torch.tensor([n - r + len(path) - 1 for (n, r), paths in zip(_seqs(c), _paths(s)) for path in paths], device="cuda")

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


def _values(x, xs):
    if xs is None:
        return x.double()
    levels = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device="cuda")
    x = torch.stack((levels[(x % 16).long()], levels[(x // 16).long()]), -1).flatten(-2)
    return x * torch.exp2(xs.double() - 127).repeat_interleave(32, -1)


def _exact_attention(s):
    """Row by row over the tokens that it sees, some rows of a sequence at a time."""
    c, out, r0 = s.c, [], 0
    nkv, hd, group = c["nkv"], c["hd"], c["nh"] // c["nkv"]
    for b, ((n, r), paths) in enumerate(zip(_seqs(c), _paths(s))):
        pages = s.pages[b, :-(-n // c["page"])].long()
        k, v = (_values(x[0][pages], xs[0][pages] if xs is not None else None).transpose(0, 1).reshape(nkv, -1, hd)[:, :n]
                for x, xs in ((s.k, s.ks), (s.v, s.vs)))
        kt = k.transpose(1, 2).contiguous()
        base = n - r
        for i in range(0, r, 16):
            some = paths[i:i + 16]
            seen = torch.zeros((len(some), n), dtype=torch.bool)
            for j, path in enumerate(some):
                last = path[-c["window"]:] if c["window"] else path
                seen[j, max(0, base + len(path) - c["window"]) if c["window"] else 0:base] = True
                seen[j, [base + a for a in last]] = True
            q = s.q[r0 + i:r0 + i + len(some)].double().view(-1, nkv, group, hd)
            a = torch.matmul(q.permute(1, 2, 0, 3).reshape(nkv, -1, hd), kt).view(nkv, group, -1, n) / math.sqrt(hd)
            a = torch.where(seen.cuda(), a, -math.inf)
            if s.sink is not None:
                a = torch.cat((a, s.sink.double().view(nkv, group, 1, 1).expand(-1, -1, len(some), 1)), -1)
            p = torch.softmax(a, -1)[..., :n].reshape(nkv, -1, n)
            out.append(torch.matmul(p, v).view(nkv, group, len(some), hd).permute(2, 0, 1, 3).reshape(len(some), -1))
        r0 += r
    return torch.cat(out)


def _exact_verify(s):
    """Sequence by sequence, as the method is told: a draft that the target likes too little is refused, what is left of the target's
    probabilities is scaled to one again, and the next draft of the same parent stands against that."""
    c, ends = s.c, s.row0.tolist()
    up, tokens, u = s.parent.tolist(), s.token.tolist(), s.u.tolist()
    n_kept, kept, after = [], [], []

    def target(r):
        if c["temp"] <= 0:
            p = torch.zeros(c["vocab"], dtype=torch.float64, device="cuda")
            p[s.logits[r].argmax()] = 1
            return p
        return torch.softmax(s.logits[r].double() / torch.tensor(c["temp"]).item(), -1)
    for a, b in zip(ends, ends[1:]):
        path, p = [0], target(a)
        for i in range(1, b - a):
            if up[a + i] != path[-1]:
                continue
            if s.q is None or c["temp"] <= 0:
                q = torch.zeros_like(p)
                q[tokens[a + i]] = 1
            else:
                q = s.q[a + path[-1]].double()
            if u[a + i] * q[tokens[a + i]] < p[tokens[a + i]]:
                path.append(i)
                p = target(a + i)
                continue
            rest = (p - q).clamp(min=0)
            p = rest / rest.sum() if rest.sum() > 0 else rest
        if not p.sum() > 0:
            p = target(a + path[-1])
        run = torch.cumsum(p, 0)
        after.append(min(int((run <= u[a] * run[-1]).sum()), c["vocab"] - 1))
        n_kept.append(len(path))
        kept.append(path + [-1] * (s.max_rows - len(path)))
    return {"n_kept": _ints(n_kept), "kept": _ints(kept), "next": _ints(after)}


def _exact_keep(s):
    """Token by token."""
    c, page = s.c, s.c["page"]
    pages, kept, n_kept = s.pages.tolist(), s.kept.tolist(), s.n_kept.tolist()
    to, frm, length = [], [], []
    for b, (n, r) in enumerate(_seqs(c)):
        for j in range(r):      # (the slots behind the kept rows as they were)
            t, f = n - r + j, n - r + (kept[b][j] if j < n_kept[b] else j)
            to.append((pages[b][t // page], t % page))
            frm.append((pages[b][f // page], f % page))
        length.append(n - r + n_kept[b])
    to, frm = torch.tensor(to, device="cuda").T, torch.tensor(frm, device="cuda").T
    if c["dt"] == "f16":
        k, v = s.k.clone(), s.v.clone()
        for x, old in ((k, s.k), (v, s.v)):
            x[:, to[0], :, to[1]] = old[:, frm[0], :, frm[1]]
        return {"k": k, "v": v, "len": _ints(length)}
    kv = [_values(x[:, frm[0], :, frm[1]], xs[:, frm[0], :, frm[1]]) for x, xs in ((s.k, s.ks), (s.v, s.vs))]   # [rows][layers][nkv][hd]
    return {"kv": torch.stack([x.transpose(0, 1).flatten(2) for x in kv], 1), "len": _ints(length)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify, "keep": _exact_keep}[case["kind"]](s)


# ------------------------------------------------------------------- work

def work(case):
    c = case
    if c["kind"] == "verify":
        # any row's probabilities may be asked for; of the drafts' own, one row of each sequence
        rows = sum(max(1, c["rows"] - i * 5 % max(1, c["rows"] // 2)) for i in range(c["seqs"]))
        return {"bytes": 4 * c["vocab"] * (rows + (c["seqs"] if c["q"] and c["temp"] > 0 else 0)) + 16 * rows, "flops": 4 * c["vocab"] * rows}
    hd, seqs = c["hd"], _seqs(c)
    token = c["nkv"] * (4 * hd if c["dt"] == "f16" else hd + hd // 16)      # k and v of one token
    rows = sum(r for _, r in seqs)
    if c["kind"] == "append":
        return {"bytes": rows * (4 * hd * (2 * c["nh"] + 2 * c["nkv"]) + 2 * token + 8 * hd * c["nkv"]), "flops": 10 * rows * hd * (c["nh"] + 2 * c["nkv"])}
    if c["kind"] == "keep":
        return {"bytes": 2 * c["layers"] * token * max(1, rows // 4), "flops": 0}      # (a path through a tree is a small part of its rows)
    seen = pairs = 0
    for n, r in seqs:
        w = c["window"] or n
        seen += min(n - r, w) + r
        pairs += r * min(n - r + 3, w)      # (some ancestors)
    return {"bytes": seen * token + 8 * rows * c["nh"] * hd, "flops": 4 * hd * c["nh"] * pairs}
