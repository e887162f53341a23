"""Oracle of the drafted-token operators in 64 bits (numpy): attention for a
tree of drafted tokens over a cache, verification against the target's
probabilities, commit of the accepted rows.  Written from the definitions in
include/moe_hip.h, node by node and token by token."""
import numpy as np


def chains(parent):
    """Each node's ancestors and itself, root first; None: no token."""
    out = []
    for i, p in enumerate(parent):
        p = int(p)
        above = [] if p == -1 else out[p] if 0 <= p < i else None
        out.append(None if above is None else above + [i])
    return out


def attend(x, w, rms, eps, cos_t, sin_t, parent, pos, kc, vc, nh, nkv, hd):
    """(y, k, v, live): y, k, v hold rows of live nodes only (others zero).
    x [B][N][d], w = (wq, wk, wv, wo), caches [B][max_seq][nkv*hd]."""
    wq, wk, wv, wo = (np.asarray(a, np.float64) for a in w)
    x64, rms = x.astype(np.float64), rms.astype(np.float64)
    B, N, d = x.shape
    S, G = kc.shape[1], nh // nkv
    y, live = np.zeros((B, N, d)), np.zeros((B, N), bool)
    kd, vd = np.zeros((B, N, nkv * hd)), np.zeros((B, N, nkv * hd))

    def rope(t, p, heads):
        t = t.reshape(heads, hd)
        c, s = cos_t[p].astype(np.float64), sin_t[p].astype(np.float64)
        a, b = t[:, 0::2].copy(), t[:, 1::2].copy()
        r = np.empty_like(t)
        r[:, 0::2], r[:, 1::2] = a * c - b * s, a * s + b * c
        return r.reshape(-1)

    for b in range(B):
        p = int(pos[b])
        if not 0 <= p < S:
            continue
        ch = chains(parent[b])
        q = np.zeros((N, nh * hd))
        for i in range(N):
            if ch[i] is None or p + len(ch[i]) - 1 >= S:
                continue
            live[b, i] = True
            at = p + len(ch[i]) - 1
            z = x64[b, i] / np.sqrt((x64[b, i] ** 2).mean() + np.float64(np.float32(eps))) * rms
            q[i], kd[b, i], vd[b, i] = rope(z @ wq, at, nh), rope(z @ wk, at, nkv), z @ wv
        for i in range(N):
            if not live[b, i]:
                continue
            K = np.concatenate((kc[b, :p].astype(np.float64), kd[b, ch[i]]))
            V = np.concatenate((vc[b, :p].astype(np.float64), vd[b, ch[i]]))
            o = np.zeros((nh, hd))
            for h in range(nh):
                lo = (h // G) * hd
                s = K[:, lo:lo + hd] @ q[i, h * hd:(h + 1) * hd] / np.sqrt(hd)
                e = np.exp(s - s.max())
                o[h] = (e / e.sum()) @ V[:, lo:lo + hd]
            y[b, i] = x64[b, i] + o.reshape(-1) @ wo
    return y, kd, vd, live


def verify(p, q, parent, token, u_accept, u_sample):
    """(path, n_acc, next) by the recursion itself: what is left of the
    target's distribution is normalised after every rejection.  p, q
    [B][N][V] (q None: looked-up drafts)."""
    B, N, V = p.shape
    path, n_acc = np.full((B, N), -1, np.int32), np.full(B, -1, np.int32)
    nxt = np.full(B, -1, np.int32)
    pos0 = lambda r: np.where(r > 0, r, 0.0)  # noqa: E731  (negatives and NaN count as 0)
    for b in range(B):
        if parent[b, 0] != -1:
            continue
        cur, n = 0, 0
        path[b, 0] = 0
        left, total = None, 1.0
        with np.errstate(invalid="ignore", over="ignore"):
            while True:
                left, total, tried, moved = p[b, cur].astype(np.float64), 1.0, False, False
                for c in range(cur + 1, N):
                    t = int(token[b, c])
                    if parent[b, c] != cur or not 0 <= t < V:
                        continue
                    drawn = np.zeros(V) if q is None else pos0(q[b, cur].astype(np.float64))
                    if q is None:
                        drawn[t] = 1.0
                    if float(u_accept[b, c]) * drawn[t] < pos0(left[t] / total):
                        cur, n, moved = c, n + 1, True
                        path[b, n] = c
                        break
                    if q is None:
                        left[t] = 0.0
                        left = pos0(left)
                    else:
                        left = pos0(left / total - drawn) if total > 0 else np.zeros(V)
                    total, tried = left.sum(), True
                if not moved:
                    break
            n_acc[b] = n
            left = pos0(left)
            if tried and left.sum() == 0:
                left = pos0(p[b, cur].astype(np.float64))
            total = left.sum()
            if not 0 < total < np.inf:
                continue
            over = np.nonzero(np.cumsum(left) > float(u_sample[b]) * total)[0]
            nxt[b] = over[0] if len(over) else np.nonzero(left)[0][-1]
    return path, n_acc, nxt


def commit(kd, vd, kc, vc, pos, path, n_acc):
    """New (kc, vc, pos) of one block."""
    kc, vc, out = kc.copy(), vc.copy(), pos.copy()
    B, S = kc.shape[:2]
    N = kd.shape[1]
    for b in range(B):
        p = int(pos[b])
        if n_acc[b] < 0 or not 0 <= p < S:
            continue
        for j in range(min(int(n_acc[b]), N - 1) + 1):
            if 0 <= path[b, j] < N and p + j < S:
                kc[b, p + j], vc[b, p + j] = kd[b, path[b, j]], vd[b, path[b, j]]
        out[b] = min(p + min(int(n_acc[b]), N - 1) + 1, S)
    return kc, vc, out
