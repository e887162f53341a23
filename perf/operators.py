"""The performance cases of libmoe_hip's operators for drafted tokens.

A serving step with drafts runs, for B sequences with a tree of N drafted
tokens each (node 0 the last token that is certain):
  attend   moe_hip_attn_tree_dev: y = x + Attn(rms_norm(x)) of every node over
           the sequence's cache and the node's ancestors; the nodes' keys and
           values go to draft buffers
  verify   moe_hip_tree_verify_dev: the accepted path and the next token from
           the target's and the draft's probabilities and given random numbers
  commit   moe_hip_tree_commit_dev: the accepted nodes' keys and values into
           the caches of every block
A case is a dict with its "kind" and sizes.  run() computes it from elementary
torch operations, or (own) through the library.
"""
import ctypes as C
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One sequence, a handful of drafted tokens: latency.
        dict(name="tree of 8, one sequence", kind="attend", B=1, N=8, ctx=1024, d=512, nh=8, nkv=2, hd=64, shape="tree"),
        # Plain decode through the same entry point: one token of 64 sequences.
        dict(name="single tokens, 64 sequences", kind="attend", B=64, N=1, ctx=1024, d=512, nh=8, nkv=2, hd=64, shape="chain"),
        # The ordinary serving step.
        dict(name="trees of 16, 64 sequences", kind="attend", B=64, N=16, ctx=1024, d=512, nh=8, nkv=2, hd=64, shape="tree"),
        # The widest trees at twice the context: the largest call.
        dict(name="trees of 64, 64 sequences", kind="attend", B=64, N=64, ctx=2048, d=512, nh=8, nkv=2, hd=64, shape="tree"),
        # Two long documents: few rows, long caches.
        dict(name="long context, two sequences", kind="attend", B=2, N=32, ctx=32768, d=512, nh=8, nkv=2, hd=64, shape="tree"),
        # Head sizes, widths, rows and a context that no tile divides.
        dict(name="ragged trees", kind="attend", B=7, N=13, ctx=777, d=320, nh=6, nkv=3, hd=40, shape="ragged"),
        # One sequence's chain of drafts, the small vocabulary: latency.
        dict(name="verify one chain", kind="verify", B=1, N=6, V=4096, shape="chain", probs=True),
        # The ordinary serving step.
        dict(name="verify trees of 16", kind="verify", B=64, N=16, V=32768, shape="tree", probs=True),
        # A large vocabulary and wide trees.
        dict(name="verify large vocabulary", kind="verify", B=64, N=32, V=131072, shape="tree", probs=True),
        # Drafts looked up rather than drawn (no draft probabilities).
        dict(name="verify looked-up drafts", kind="verify", B=33, N=24, V=50001, shape="ragged", probs=False),
        # The eight blocks' caches after one sequence's step.
        dict(name="commit one sequence", kind="commit", B=1, N=8, ctx=1024, blocks=8, kd=128),
        # And after the serving step.
        dict(name="commit 64 sequences", kind="commit", B=64, N=16, ctx=256, blocks=8, kd=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "commit"])
    shape = rng.choice(["tree", "tree", "chain", "ragged"])
    while True:
        if kind == "attend":
            hd = 8 * rng.randint(1, 8) if rng.random() < 0.5 else rng.choice([32, 64])
            nkv = rng.choice([1, 2, 3, 4, 8])
            c = dict(kind=kind, B=_log(rng, 1, 96), N=_log(rng, 1, 64), ctx=_log(rng, 1, 32768), d=4 * _log(rng, 16, 256),
                     nh=nkv * rng.randint(1, 8), nkv=nkv, hd=hd, shape=shape)
            if c["B"] * c["ctx"] * nkv * hd * 8 > 6e8 or work(c)["flops"] > 2.2e10 or c["nh"] * hd > 1024:
                continue
            # (the plain form holds every score)
            if c["B"] * c["N"] * c["nh"] * (c["ctx"] + c["N"]) > 7e7:
                continue
        elif kind == "verify":
            c = dict(kind=kind, B=_log(rng, 1, 128), N=_log(rng, 1, 64), V=_log(rng, 16, 131072), shape=shape, probs=rng.random() < 0.7)
            if c["B"] * c["N"] * c["V"] > 2.6e8:
                continue
        else:
            c = dict(kind=kind, B=_log(rng, 1, 96), N=_log(rng, 1, 64), ctx=_log(rng, 1, 1024), blocks=rng.randint(1, 16), kd=8 * _log(rng, 1, 64))
            if c["B"] * (c["ctx"] + c["N"]) * c["blocks"] * c["kd"] > 4e7:
                continue
        return c


# ---------------------------------------------------------------------- inputs
def _gen(seed, salt, device="cuda"):
    return torch.Generator(device=device).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _randn(seed, salt, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=_gen(seed, salt))


def _rand(seed, salt, *shape):
    return torch.rand(*shape, device="cuda", dtype=torch.float32, generator=_gen(seed, salt))


def _parents(case, seed):
    """Chains, trees (each node hangs on one of the four nodes before its
    half, so trees are a few levels deep with up to a dozen children a node),
    or trees with fewer nodes than N (the others are no tokens: -2)."""
    B, N = case["B"], case["N"]
    i = torch.arange(N).unsqueeze(0).expand(B, N)
    if case["shape"] == "chain":
        return (i - 1).int().contiguous()
    g = _gen(seed, 1, "cpu")
    r = torch.randint(0, 4, (B, N), generator=g)
    parent = torch.clamp(torch.minimum((i - 1) // 2 - r + 1, i - 1), min=0)
    parent[:, 0] = -1
    if case["shape"] == "ragged":
        used = torch.randint(1, N + 1, (B, 1), generator=g)
        parent = torch.where(i < used, parent, torch.full_like(parent, -2))
    return parent.int().contiguous()


def _positions(case, seed):
    """Most sequences at the full context, the others somewhere before it."""
    B, ctx = case["B"], case["ctx"]
    g = _gen(seed, 2, "cpu")
    pos = torch.full((B,), ctx, dtype=torch.int32)
    early = torch.rand(B, generator=g) < 0.25
    early[0] = False
    return torch.where(early, torch.randint(0, ctx + 1, (B,), generator=g, dtype=torch.int32), pos)


def _rope(max_seq, hd):
    i = np.arange(hd // 2, dtype=np.float64)
    ang = np.arange(max_seq)[:, None] / 10000.0 ** (2 * i / hd)[None, :]
    return torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))


_STREAM = []


def _stream():
    """The program's compute stream: the library's calls share one workspace,
    so they are queued on one stream."""
    if not _STREAM:
        _STREAM.append(torch.cuda.Stream())
    return _STREAM[0]


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import moe_hip
    return moe_hip


class State:
    """What a program keeps between calls."""


def _attend_inputs(case, seed):
    B, N, d, nh, nkv, hd = (case[k] for k in ("B", "N", "d", "nh", "nkv", "hd"))
    S = case["ctx"] + N
    shapes = ((d, nh * hd), (d, nkv * hd), (d, nkv * hd), (nh * hd, d))
    # (queries three times as long as keys: each attends a few positions, not all alike)
    w = [(3.0 if j == 0 else 1.0) * _randn(seed, 10 + j, *s) / math.sqrt(s[0]) for j, s in enumerate(shapes)]
    cache = [_randn(seed, 20 + j, B, S, nkv * hd) for j in range(2)]
    rms = 1.0 + 0.1 * _randn(seed, 6, d)
    return _randn(seed, 5, B, N, d), w, rms, cache, _rope(S, hd), _parents(case, seed), _positions(case, seed)


def _verify_inputs(case, seed):
    """The target's softmax of N(0, 2) logits and the draft's, which is near it
    but not the same; a child's token is a draw from its parent's draft
    distribution, u are uniform."""
    B, N, V = case["B"], case["N"], case["V"]
    parent = _parents(case, seed)
    up = parent.long().clamp(min=0).cuda()
    z = 2.0 * _randn(seed, 30, B, N, V)
    p = torch.softmax(z, 2)
    z = 0.8 * z + 0.6 * _randn(seed, 31, B, N, V)
    q = torch.softmax(z, 2)
    # (a draw of softmax(z) is the largest z plus Gumbel noise)
    noise = _rand(seed, 32, B, N, V).clamp_(1e-12, 1.0 - 1e-7).log_().neg_().log_().neg_()
    b = torch.arange(B, device="cuda").unsqueeze(1)
    token = noise.add_(z[b, up]).argmax(2).int()
    return p, q if case["probs"] else None, parent, token, _rand(seed, 33, B, N), _rand(seed, 34, B)


def _commit_inputs(case, seed):
    """Accepted paths of every length: node 0, then rising node indices."""
    B, N = case["B"], case["N"]
    g = _gen(seed, 3, "cpu")
    n_acc = torch.randint(0, (N + 1) // 2, (B,), generator=g)
    order = torch.rand(B, N, generator=g)
    order[:, 0] = -1.0
    rank = order.argsort(1).argsort(1)
    keep = torch.sort(torch.where(rank <= n_acc.unsqueeze(1), torch.arange(N).unsqueeze(0), torch.full((B, N), N)), 1).values
    path = torch.where(keep < N, keep, torch.full_like(keep, -1)).int()
    L, S, kd = case["blocks"], case["ctx"] + N, case["kd"]
    cache = [_randn(seed, 40 + j, L, B, S, kd) for j in range(2)]
    draft = [_randn(seed, 42 + j, L, B, N, kd) for j in range(2)]
    return cache, draft, _positions(case, seed), path.contiguous(), n_acc.int()


def prepare(case, seed):
    s = State()
    s.case, kind, s.stream = case, case["kind"], _stream()
    if kind == "attend":
        s.x, s.w, s.rms, s.cache, rope, parent, pos = _attend_inputs(case, seed)
        B, N, kd = case["B"], case["N"], case["nkv"] * case["hd"]
        s.rope = [t.cuda() for t in rope]
        s.parent, s.pos = parent.cuda(), pos.cuda()
        s.y, s.kd, s.vd = torch.zeros_like(s.x), torch.zeros(B, N, kd, device="cuda"), torch.zeros(B, N, kd, device="cuda")
        if own:
            mh = _library()
            s.attn = mh.Attn(case["d"], case["nh"], case["nkv"], case["hd"], case["ctx"] + N)
            s.attn.load(*[w.cpu().numpy() for w in s.w], s.rms.cpu().numpy())
            s.attn.set_rope(*[t.numpy() for t in rope])
    elif kind == "verify":
        s.p, s.q, parent, s.token, s.u_accept, s.u_sample = _verify_inputs(case, seed)
        s.parent = parent.cuda()
        B, N = case["B"], case["N"]
        s.path, s.n_acc, s.next = (torch.empty(*sh, dtype=torch.int32, device="cuda") for sh in ((B, N), (B,), (B,)))
    else:
        s.cache, s.draft, pos, path, n_acc = _commit_inputs(case, seed)
        s.pos, s.path, s.n_acc = pos.cuda(), path.cuda(), n_acc.cuda()
        s.pos_out = torch.empty_like(s.pos)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- plain form
def _depth_and_ancestors(parent):
    """live [B][N], depth [B][N] and seen [B][N][N] (j is i or above it): the
    boolean closure of the parent relation by squaring."""
    B, N = parent.shape
    j = torch.arange(N, device=parent.device)
    link = (parent.unsqueeze(2) == j) & (j < j.unsqueeze(1))
    seen = (link | torch.eye(N, dtype=torch.bool, device=parent.device)).float()
    for _ in range(max(1, (N - 1).bit_length())):
        seen = (torch.matmul(seen, seen) > 0).float()
    roots = (parent == -1).float()
    live = torch.matmul(seen, roots.unsqueeze(2)).squeeze(2) > 0
    return live, seen.sum(2).long() - 1, seen > 0


def _rotate(v, cos, sin, heads):
    """v [B][N][heads * hd], cos and sin [B][N][hd / 2]."""
    B, N, w = v.shape
    v = v.reshape(B, N, heads, w // heads // 2, 2)
    a, b, c, s = v[..., 0], v[..., 1], cos.unsqueeze(2), sin.unsqueeze(2)
    return torch.stack((a * c - b * s, a * s + b * c), -1).reshape(B, N, w)


def _plain_attend(s):
    case = s.case
    B, N, nh, nkv, hd = (case[k] for k in ("B", "N", "nh", "nkv", "hd"))
    G, S = nh // nkv, s.cache[0].shape[1]
    live, depth, seen = _depth_and_ancestors(s.parent)
    at = s.pos.long().unsqueeze(1) + depth
    live = live & (at < S)
    cos, sin = (t[at.clamp(max=S - 1)] for t in s.rope)
    xn = s.x * torch.rsqrt(s.x.square().mean(2, keepdim=True) + EPS) * s.rms
    wq, wk, wv, wo = s.w
    q, k, v = _rotate(xn @ wq, cos, sin, nh), _rotate(xn @ wk, cos, sin, nkv), xn @ wv

    def heads(t):  # [B][rows][nkv * hd] -> [B][nkv][rows][hd]
        return t.reshape(B, -1, nkv, hd).transpose(1, 2).contiguous()

    qh = q.reshape(B, N, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * N, hd)
    kh, vh = (torch.cat((heads(c), heads(t)), 2) for c, t in zip(s.cache, (k, v)))
    scores = torch.matmul(qh, kh.transpose(2, 3)).reshape(B, nkv, G, N, S + N) / math.sqrt(hd)
    cached = (torch.arange(S, device="cuda") < s.pos.unsqueeze(1)).unsqueeze(1).expand(B, N, S)
    mask = torch.cat((cached, seen), 2).unsqueeze(1).unsqueeze(1)
    scores = scores.masked_fill(~mask, -math.inf)
    e = torch.exp(scores - scores.amax(4, keepdim=True))
    e = (e / e.sum(4, keepdim=True)).reshape(B, nkv, G * N, S + N)
    o = torch.matmul(e, vh).reshape(B, nkv, G, N, hd).permute(0, 3, 1, 2, 4).reshape(B, N, nh * hd)
    keep = live.unsqueeze(2)
    return {"y": torch.where(keep, s.x + o @ wo, s.y), "k": torch.where(keep, k, s.kd), "v": torch.where(keep, v, s.vd)}


def _plain_verify(s):
    """In 64 bits: the outputs are whole numbers that follow from comparisons
    of long sums.  The walk is a sequence of decisions, each of which hangs on
    the one before: children come after their parents, so one pass over the
    nodes in order is the whole of it."""
    B, N, V = s.p.shape
    b = torch.arange(B, device="cuda")
    parent, token = s.parent.long(), s.token.long()
    cur = torch.zeros(B, dtype=torch.long, device="cuda")
    n = torch.zeros_like(cur)
    path = torch.full((B, N + 1), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    a = torch.zeros(B, dtype=torch.float64, device="cuda")
    w = torch.ones_like(a)
    gone = torch.zeros(B, V, dtype=torch.bool, device="cuda")

    def left(a, gone):
        row = s.p[b, cur].double()
        if s.q is None:
            return torch.where(gone, 0.0, row)
        return torch.clamp(row - a.unsqueeze(1) * s.q[b, cur].double(), min=0.0)

    for i in range(1, N):
        t, here = token[:, i], parent[:, i] == cur
        u, pt = s.u_accept[:, i].double(), s.p[b, cur, t].double()
        if s.q is None:
            yes = here & (u * w < torch.where(gone[b, t], 0.0, pt))
        else:
            qt = s.q[b, cur, t].double()
            yes = here & (u * qt * w < torch.clamp(pt - a * qt, min=0.0))
        no = here & ~yes
        gone = gone & ~yes.unsqueeze(1)
        gone[b, t] = gone[b, t] | no
        a = torch.where(no, a + w, a)
        w = torch.where(no, left(a, gone).sum(1), w)
        n = torch.where(yes, n + 1, n)
        path[b, torch.where(yes, n, N)] = i
        cur = torch.where(yes, i, cur)
        a, w = torch.where(yes, 0.0, a), torch.where(yes, 1.0, w)
    row = left(a, gone)
    empty = row.sum(1, keepdim=True) == 0.0
    row = torch.where(empty, s.p[b, cur].double(), row)
    cum = torch.cumsum(row, 1)
    nxt = (cum <= (s.u_sample.double() * row.sum(1)).unsqueeze(1)).sum(1)
    last = V - 1 - (row > 0).flip(1).int().argmax(1)
    return {"path": path[:, :N].int(), "n_acc": n.int(), "next": torch.minimum(nxt, last).int()}


def _plain_commit(s):
    B, N = s.path.shape
    b = torch.arange(B, device="cuda").unsqueeze(1)
    rows = s.pos.long().unsqueeze(1) + torch.arange(N, device="cuda")
    take = (s.path >= 0).unsqueeze(2)
    frm = s.path.long().clamp(min=0)
    k, v = ((c, t[:, b, frm]) for c, t in zip(s.cache, s.draft))
    k[0][:, b, rows] = torch.where(take, k[1], k[0][:, b, rows])
    v[0][:, b, rows] = torch.where(take, v[1], v[0][:, b, rows])
    return {"k": s.cache[0], "v": s.cache[1], "pos": s.pos + s.n_acc + 1}


# -------------------------------------------------------------------------- run
def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def run(s):
    case, kind = s.case, s.case["kind"]
    if not own:
        with torch.cuda.stream(s.stream):
            return {"attend": _plain_attend, "verify": _plain_verify, "commit": _plain_commit}[kind](s)
    mh, st = _library(), C.c_void_p(s.stream.cuda_stream)
    B, N = case["B"], case["N"]
    if kind == "attend":
        s.attn.tree_dev(_ptr(s.x), _ptr(s.y), B, N, _ptr(s.parent), _ptr(s.pos), _ptr(s.cache[0]), _ptr(s.cache[1]), _ptr(s.kd),
                        _ptr(s.vd), EPS, st)
        return {"y": s.y, "k": s.kd, "v": s.vd}
    if kind == "verify":
        V = case["V"]
        mh.tree_verify_dev(_ptr(s.p), V, _ptr(s.q), V, B, N, V, _ptr(s.parent), _ptr(s.token), _ptr(s.u_accept), _ptr(s.u_sample),
                           _ptr(s.path), _ptr(s.n_acc), _ptr(s.next), st)
        return {"path": s.path, "n_acc": s.n_acc, "next": s.next}
    ptrs = [[t[i].data_ptr() for i in range(case["blocks"])] for t in (*s.draft, *s.cache)]
    mh.tree_commit_dev(*ptrs, B, N, case["kd"], case["ctx"] + N, _ptr(s.pos), _ptr(s.path), _ptr(s.n_acc), _ptr(s.pos_out), st)
    return {"k": s.cache[0], "v": s.cache[1], "pos": s.pos_out}


# ------------------------------------------------------------------------- work
def work(case):
    """Every input that the outputs hang on read once, every output written
    once.  Contexts: three quarters of the sequences at ctx, the others at
    half of it on average."""
    kind, B, N = case["kind"], case["B"], case["N"]
    live = 0.5 * (N + 1) if case.get("shape") == "ragged" else float(N)
    if kind == "attend":
        d, qd, kd = case["d"], case["nh"] * case["hd"], case["nkv"] * case["hd"]
        ctx, rows = 0.875 * case["ctx"], B * live
        proj = 2.0 * d * (qd + kd)
        return {"bytes": 4.0 * (proj + 2.0 * B * ctx * kd + rows * (2 * d + 2 * kd)), "flops": rows * (2.0 * proj + 4.0 * qd * (ctx + 1.0))}
    if kind == "verify":
        # (the row that the last decision of a sequence hangs on)
        return {"bytes": 4.0 * B * (case["V"] * (2 if case["probs"] else 1) + 4 * N), "flops": 3.0 * B * case["V"]}
    rows = 1.0 + 0.5 * ((N + 1) // 2 - 1)
    return {"bytes": 4.0 * (4.0 * case["blocks"] * B * rows * case["kd"] + B * (N + 3)), "flops": 0.0}


# ------------------------------------------------------------------------ exact
def exact(case, seed):
    return {"attend": _exact_attend, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](case, seed)


def _chains(parent):
    """Each node's ancestors and itself, root first (None: no token)."""
    out = []
    for row in parent.tolist():
        chains = []
        for i, p in enumerate(row):
            above = [] if p == -1 else chains[p] if 0 <= p < i else None
            chains.append(None if above is None else above + [i])
        out.append(chains)
    return out


def _exact_attend(case, seed):
    B, N, d, nh, nkv, hd = (case[k] for k in ("B", "N", "d", "nh", "nkv", "hd"))
    x, (wq, wk, wv, wo), rms, cache, rope, parent, pos = _attend_inputs(case, seed)
    S, G = case["ctx"] + N, nh // nkv
    x, wq, wk, wv, wo, rms = (t.double() for t in (x, wq, wk, wv, wo, rms))
    cos, sin = (t.double().cuda() for t in rope)
    xn = x / torch.sqrt((x * x).sum(2, keepdim=True) / d + float(np.float32(EPS))) * rms
    chains = _chains(parent)
    y, kd, vd = torch.zeros_like(x), torch.zeros(B, N, nkv * hd, device="cuda").double(), torch.zeros(B, N, nkv * hd, device="cuda").double()

    def turn(v, at, heads):
        v = v.reshape(v.shape[0], heads, hd // 2, 2)
        c, t = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
        return torch.stack((v[..., 0] * c - v[..., 1] * t, v[..., 0] * t + v[..., 1] * c), 3).reshape(v.shape[0], heads, hd)

    for b in range(B):
        p = int(pos[b])
        on = [i for i in range(N) if chains[b][i] is not None and p + len(chains[b][i]) - 1 < S]
        if not on:
            continue
        at = torch.tensor([p + len(chains[b][i]) - 1 for i in on], device="cuda")
        rows = torch.tensor(on, device="cuda")
        z = xn[b, rows]
        q, k, v = turn(z @ wq, at, nh), turn(z @ wk, at, nkv), (z @ wv).reshape(len(on), nkv, hd)
        kd[b, rows], vd[b, rows] = k.reshape(len(on), -1), v.reshape(len(on), -1)
        see = torch.tensor([[j in chains[b][i] for j in on] for i in on], device="cuda").repeat_interleave(G, 0)
        o = torch.empty(len(on), nh, hd, dtype=torch.float64, device="cuda")
        for h in range(nkv):
            kk = torch.cat((cache[0][b, :p, h * hd:(h + 1) * hd].double(), k[:, h]), 0)
            vv = torch.cat((cache[1][b, :p, h * hd:(h + 1) * hd].double(), v[:, h]), 0)
            sc = q[:, h * G:(h + 1) * G].reshape(-1, hd) @ kk.T.contiguous() / math.sqrt(hd)
            sc[:, p:][~see] = -math.inf
            o[:, h * G:(h + 1) * G] = (torch.softmax(sc, 1) @ vv).reshape(len(on), G, hd)
        y[b, rows] = x[b, rows] + o.reshape(len(on), -1) @ wo
    return {"y": y, "k": kd, "v": vd}


def _exact_verify(case, seed):
    """Sequence by sequence from the textbook recursion: the distribution that
    is left is normalised again after every rejection."""
    p, q, parent, token, ua, us = _verify_inputs(case, seed)
    N = case["N"]
    kids, token, ua, us = parent.tolist(), token.tolist(), ua.double().tolist(), us.double().tolist()
    paths, counts, nexts = [], [], []
    for b in range(case["B"]):
        cur, path = 0, [0]
        while True:
            left, moved = p[b, cur].double(), False
            fresh = left
            for c in [i for i in range(cur + 1, N) if kids[b][i] == cur]:
                t = token[b][c]
                drawn = q[b, cur].double() if q is not None else torch.zeros_like(left).index_fill_(0, torch.tensor([t], device="cuda"), 1.0)
                if ua[b][c] * float(drawn[t]) < float(left[t]):
                    cur, moved = c, True
                    path.append(c)
                    break
                rest = torch.clamp(left - drawn, min=0.0)
                total = float(rest.sum())
                left = rest / total if total > 0 else rest
            if not moved:
                break
        if float(left.sum()) == 0.0:
            left = fresh
        cum = torch.cumsum(left, 0)
        nexts.append(min(int((cum <= us[b] * float(left.sum())).sum()), int(left.nonzero().max())))
        paths.append(path + [-1] * (N - len(path)))
        counts.append(len(path) - 1)
    return {"path": torch.tensor(paths, dtype=torch.int32), "n_acc": torch.tensor(counts, dtype=torch.int32), "next": torch.tensor(nexts, dtype=torch.int32)}


def _exact_commit(case, seed):
    cache, draft, pos, path, n_acc = _commit_inputs(case, seed)
    for b in range(case["B"]):
        n, at = int(n_acc[b]) + 1, int(pos[b])
        for c, t in zip(cache, draft):
            c[:, b, at:at + n] = t[:, b, path[b, :n].long().cuda()]
    return {"k": cache[0], "v": cache[1], "pos": (pos + n_acc + 1).cuda()}
