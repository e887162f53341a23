"""Drafted tokens: attention for trees over a cache, verification, commit.

The oracle (oracle/tree_oracle.py) is the definition in 64 bits.  CPU: the
oracle against closed forms (the rule's output distribution is the target's;
a chain is successive decode steps), and the refusals.  GPU: every entry
point against the oracle.

Tolerances, attention: fp32 sums of up to 1024 products, then a softmax of
scores up to ~20 (their rounding, 2^-24 of 20 in each of the two products'
sums, moves an exponential by ~3e-6 at worst and 3e-7 in the mean): the
layer tolerance, relative 2-norm 1e-5 and 1e-4 at most, as for the decode
step.  Verification and commit: equal."""
import ctypes as C
import itertools
import os

import numpy as np
import pytest

import moe_hip as mh
import orc
import tree_oracle as to
from test_attention import make_case

EPS = 1e-5


def make_parents(kind, B, N, seed):
    rng = np.random.default_rng(seed)
    par = np.full((B, N), -2, np.int32)
    for b in range(B):
        for i in range(N):
            if kind == "chain":
                par[b, i] = i - 1
            elif kind == "star":
                par[b, i] = 0 if i else -1
            elif kind == "forest":      # several nodes hang on the context itself
                par[b, i] = rng.integers(-1, i) if i else -1
            else:
                par[b, i] = rng.integers(max(0, i - 5), i) if i else -1
        if kind == "holes":             # no tokens among them, in every form
            for i in rng.integers(0, N, max(1, N // 4)):
                par[b, i] = rng.choice([-2, i, i + 1, N, 99, -2147483648, 2147483647])
        if kind == "none" or (kind == "ragged" and b % 3 == 0):
            par[b, rng.integers(0, N) if kind == "ragged" else 0:] = -2
    return par


# ------------------------------------------------------------------------ CPU
def test_oracle_output_distribution():
    """Two children drawn from q, one node: summed over the draws and over
    both acceptances, the next token is distributed as p (the rule's purpose),
    and without q (fixed children) too."""
    rng = np.random.default_rng(1)
    for V in (2, 3, 5):
        p, q = rng.dirichlet(np.ones(V)), rng.dirichlet(np.ones(V))
        got = np.zeros(V)
        for t in itertools.product(range(V), repeat=2):
            weight, left = q[t[0]] * q[t[1]], p.copy()
            for c in t:
                a = min(1.0, left[c] / q[c])
                got[c] += weight * a
                weight *= 1 - a
                rest = np.maximum(left - q, 0)
                left = rest / rest.sum() if rest.sum() > 0 else left
            got += weight * left
        assert np.allclose(got, p, atol=1e-12)


def test_oracle_verify_closed_form():
    """The recursion equals its closed form r_j = max(p - a_j q, 0), a_{j+1} =
    a_j + sum r_j."""
    rng = np.random.default_rng(2)
    for _ in range(50):
        p, q = rng.dirichlet(np.ones(12)), rng.dirichlet(np.ones(12))
        left, a, w = p.copy(), 0.0, 1.0
        for _ in range(4):
            left = np.maximum(left - q, 0)
            left /= left.sum()
            a += w
            r = np.maximum(p - a * q, 0)
            w = r.sum()
            assert np.allclose(r / w, left, rtol=1e-7, atol=1e-9)


def test_oracle_chain_is_decode_steps():
    """A chain's rows are the decode oracle's successive steps."""
    x, w, kc, vc, pos, c, s = make_case(2, 40, [7, 20], 3)
    N, nh, nkv, hd = 5, 8, 2, 16
    rng = np.random.default_rng(4)
    xs = rng.standard_normal((2, N, x.shape[1])).astype(np.float32)
    y, kd, vd, live = to.attend(xs, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s,
                                make_parents("chain", 2, N, 0), pos, kc, vc, nh, nkv, hd)
    assert live.all()
    for i in range(N):
        xo, kc, vc = orc.attn_decode(xs[:, i].copy(), w["rms"], EPS, w["wq"], w["wk"], w["wv"],
                                     w["wo"], c, s, kc, vc, pos + i, nh, nkv, hd)
        assert orc.rel_l2(xo, y[:, i]) < 1e-6
        for b in range(2):
            assert orc.rel_l2(kc[b, pos[b] + i], kd[b, i]) < 1e-6


def test_refusals_without_gpu():
    """Arguments are checked before anything touches a device."""
    L, P = mh.lib(), C.c_void_p
    one = P(4096)
    assert L.moe_hip_attn_tree_dev(None, one, one, 1, 1, one, one, one, one, one, one, EPS, None) == 1
    assert L.moe_hip_tree_block_dev(None, None, one, one, 1, 1, one, one, one, one, one, one, EPS,
                                    None, None, None) == 1

    def verify(p=one, ldp=8, q=one, ldq=8, B=1, N=4, V=8, rest=(one,) * 7):
        return L.moe_hip_tree_verify_dev(p, ldp, q, ldq, B, N, V, *rest, None)

    assert verify(B=0) == 0
    assert verify(B=-1) == 1 and verify(N=0) == 1 and verify(N=65) == 1 and verify(V=0) == 1
    assert verify(ldp=7) == 1 and verify(ldq=7) == 1 and verify(p=None) == 1
    assert verify(B=1 << 20, N=2) == 2
    assert verify(V=(1 << 30) + 1, ldp=1 << 31, ldq=1 << 31) == 2
    for i in range(7):
        assert verify(rest=tuple(None if j == i else one for j in range(7))) == 1

    def commit(n=1, ptrs=None, B=1, N=2, kd=16, S=8, pos=P(1 << 20), path=one, n_acc=one, out=None):
        ptrs = ptrs or [[0x10000], [0x20000], [0x30000], [0x40000]]
        arrs = [(P * max(1, len(v)))(*v) for v in ptrs]
        return L.moe_hip_tree_commit_dev(n, *arrs, B, N, kd, S, pos, path, n_acc, out, None)

    assert commit(B=0) == 0
    assert commit(n=-1) == 1 and commit(S=0) == 1 and commit(N=65) == 1 and commit(B=-1) == 1
    assert commit(kd=6) == 2 and commit(kd=0) == 2
    assert commit(pos=None) == 1 and commit(path=None) == 1 and commit(n_acc=None) == 1
    assert commit(ptrs=[[0x10008], [0x20000], [0x30000], [0x40000]]) == 1      # alignment
    assert commit(ptrs=[[0x10000], [0x20000], [0x30000], [None]]) == 1
    assert commit(ptrs=[[0x30010], [0x20000], [0x30000], [0x40000]]) == 1      # overlap
    assert commit(B=4, out=P((1 << 20) + 4)) == 1                              # part of pos
    with pytest.raises(ValueError):
        mh.tree_commit_dev([1], [1], [1], [1, 2], 1, 1, 16, 8, one, one, one)


def test_refusals_of_overlaps_without_gpu():
    """What a call writes must be apart from its other arrays."""
    L, P = mh.lib(), C.c_void_p
    B, N, V = 4, 8, 64
    at = dict(p=0x100000, q=0x200000, parent=0x300000, token=0x300100, ua=0x300200, us=0x300300,
              path=0x400000, n_acc=0x400100, next=0x400200)

    def verify(**kw):
        a = {k: P(v) for k, v in {**at, **kw}.items()}
        return L.moe_hip_tree_verify_dev(a["p"], V, a["q"], V, B, N, V, a["parent"], a["token"],
                                         a["ua"], a["us"], a["path"], a["n_acc"], a["next"], None)

    for out in ("path", "n_acc", "next"):
        for other in at:
            if other != out:
                assert verify(**{out: at[other]}) == 1, (out, other)
    assert verify(path=at["p"] + 4 * (B * N * V - 1)) == 1          # the last probability
    assert verify(next=at["n_acc"] + 12) == 1                       # the last sequence's count

    def commit(kc, vc, kd=(0x10000, 0x20000), out=None):
        arrs = [(P * 2)(*v) for v in (kd, (0x30000, 0x40000), kc, vc)]
        return L.moe_hip_tree_commit_dev(2, *arrs, 1, 2, 16, 8, P(0x1000), P(0x2000), P(0x3000),
                                         P(out) if out else None, None)

    assert commit((0x50000, 0x50000), (0x70000, 0x80000)) == 1      # one cache for two blocks
    assert commit((0x50000, 0x60000), (0x70000, 0x50010)) == 1
    assert commit((0x50000, 0x60000), (0x70000, 0x60000)) == 1      # keys and values
    assert commit((0x50000, 0x60000), (0x70000, 0x80000), kd=(0x10000, 0x50010)) == 1
    assert commit((0x50000, 0x60000), (0x70000, 0x80000), out=0x3000) == 1
    assert commit((0x50000, 0x60000), (0x70000, 0x80000), out=0x2004) == 1


# ------------------------------------------------------------------------ GPU
dev = lambda a: mh.DeviceArray.from_host(np.ascontiguousarray(a))  # noqa: E731


def run_tree(x, w, kc, vc, pos, c, s, parent, nh, nkv, hd, in_place=False, fill=7.0, at=None):
    """(y, k_draft, v_draft, caches) of one call; outputs start as `fill`."""
    B, N, d = x.shape
    own = at is None
    if own:
        at = mh.Attn(d, nh, nkv, hd, kc.shape[1])
        at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
        at.set_rope(c, s)
    try:
        dx, dk, dv, dpar, dpos = dev(x), dev(kc), dev(vc), dev(parent), dev(np.asarray(pos, np.int32))
        dy = dx if in_place else dev(np.full(x.shape, fill, np.float32))
        gk = dev(np.full((B, N, nkv * hd), fill, np.float32))
        gv = dev(np.full((B, N, nkv * hd), fill, np.float32))
        at.tree_dev(dx.ptr, dy.ptr, B, N, dpar.ptr, dpos.ptr, dk.ptr, dv.ptr, gk.ptr, gv.ptr, EPS)
        out = dy.to_host(), gk.to_host(), gv.to_host()
        assert np.array_equal(dk.to_host(), kc, equal_nan=True) and np.array_equal(dv.to_host(), vc, equal_nan=True)
        if not in_place:
            assert np.array_equal(dx.to_host(), x, equal_nan=True)
        return out
    finally:
        if own:
            at.close()


def check_tree(x, w, kc, vc, pos, c, s, parent, nh, nkv, hd, fill=7.0, **kw):
    got = run_tree(x, w, kc, vc, pos, c, s, parent, nh, nkv, hd, fill=fill, **kw)
    *want, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, parent,
                            pos, kc, vc, nh, nkv, hd)
    start = (x, None, None) if kw.get("in_place") else (None,) * 3
    for name, g, o, st in zip("ykv", got, want, start):
        kept = st[~live] if st is not None else np.full_like(g[~live], fill)
        assert np.array_equal(g[~live], kept, equal_nan=True), f"{name}: rows that are no token changed"
        if live.any():
            rel = orc.rel_l2(g[live], o[live])
            mabs = float(np.abs(g[live] - o[live]).max() / max(1.0, np.abs(o[live]).max()))
            print(f"[gpu-test]   {name} rel-L2 {rel:.2e} max {mabs:.2e}", flush=True)
            assert rel <= 1e-5 and mabs <= 1e-4, name
    return got, live


@pytest.fixture(params=["few", "many"])
def positions(request):
    """Caches as small as the case asks for, or with so many more positions
    (NaN, no sequence reaches them) that the call counts as a large one, whose
    query rows are taken in larger blocks."""
    return request.param


def tree_case(B, N, d, nh, nkv, hd, max_seq, pos, seed, kind, positions="few"):
    _, w, kc, vc, pos, c, s = make_case(B, max_seq, pos, seed, d, nh, nkv, hd)
    if positions == "many" and N * nh // nkv > 16:
        total = max(max_seq, -(-(1 << 22) // (B * N * nh)))
        kc, vc = (np.concatenate((t, np.full((B, total - max_seq, nkv * hd), np.nan, np.float32)), 1) for t in (kc, vc))
        c, s = orc.rope_tables(total, hd, 10000.0)
    w["wq"] = (2.0 * w["wq"]).astype(np.float32)    # (peaked softmax)
    x = np.random.default_rng(seed + 1).standard_normal((B, N, d)).astype(np.float32)
    return x, w, kc, vc, pos, c, s, make_parents(kind, B, N, seed)


SHAPES = [  # B, N, d, nh, nkv, hd, max_seq
    (1, 1, 64, 2, 1, 8, 4), (2, 3, 64, 2, 2, 16, 40), (3, 8, 128, 8, 2, 16, 100),
    (5, 13, 320, 6, 3, 40, 130), (2, 64, 128, 8, 1, 32, 300), (4, 16, 512, 8, 2, 64, 600),
    (3, 33, 100, 3, 3, 24, 70), (2, 17, 256, 10, 2, 48, 90), (2, 20, 192, 7, 1, 56, 65),
    (70, 1, 256, 8, 2, 64, 200), (9, 2, 1024, 16, 4, 64, 50), (1, 64, 512, 8, 2, 64, 1500),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "tree", "forest", "holes", "ragged"])
@pytest.mark.parametrize("shape", SHAPES, ids=["_".join(map(str, s)) for s in SHAPES])
def test_attn_tree(shape, kind, positions):
    """Every head size, odd widths and rows, contexts on both sides of the
    16-position tiles, trees of every form; caches untouched, rows that are no
    token left as they were."""
    B, N, d, nh, nkv, hd, S = shape
    print(f"[gpu-test] tree {shape} {kind}", flush=True)
    edge = [0, 1, 15, 16, 17, S - 1, S // 2, 31, 64, S - 2, 33]
    pos = [max(0, min(S - 1, edge[(i + len(kind)) % len(edge)])) for i in range(B)]
    case = tree_case(B, N, d, nh, nkv, hd, S, pos, 10 + N, kind, positions)
    check_tree(*case, nh, nkv, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", range(8, 65, 8))
@pytest.mark.parametrize("n_g", [(5, 3), (11, 2), (16, 4), (9, 7), (50, 4)], ids=lambda v: f"{v[0]}x{v[1]}")
def test_attn_tree_head_sizes(hd, n_g, positions):
    """Every head size with 15 to 200 query rows per kv head: each of the
    attention's block sizes, full and not."""
    N, G = n_g
    print(f"[gpu-test] tree hd {hd} rows {N * G}", flush=True)
    check_tree(*tree_case(2, N, 64, 2 * G, 2, hd, 90, [70, 33], 60 + hd, "tree", positions), 2 * G, 2, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 12, 16, 40])
def test_attn_tree_infinite_keys(N, positions):
    """A cached key with an infinite entry: its score is minus infinity
    (weight 0) or infinity (NaN) by the query's sign there, as the definition
    has it; keys above bfloat16's range are ordinary numbers."""
    B, nh, nkv, hd, S = 3, 8, 2, 16, 60
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 64, nh, nkv, hd, S, [50, 20, 41], 99, "tree", positions)
    kc[0, 7, 3] = np.inf
    kc[1, 19, 20] = -np.inf
    kc[2, 40, 5] = 3.4e38
    w["wq"][:, 5::16] = 0.0                  # (dimensions 4 and 5 turn together)
    w["wq"][:, 4::16] = 0.0
    vc[2, 8, 9] = -3.4e38
    vc[2, 8, 25] = 3.39e38
    y, _, _ = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd)
    with np.errstate(invalid="ignore"):
        o, _, _, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par,
                                  pos, kc, vc, nh, nkv, hd)
    print(f"[gpu-test] infinite keys: {np.isnan(o).any(2).mean():.2f} of the rows NaN", flush=True)
    assert live.sum() > 2 * N and np.array_equal(np.isnan(y[live]), np.isnan(o[live]))
    fine = live & ~np.isnan(o).any(2)        # (the others stand past the cache's end)
    for b in range(B):
        if fine[b].any():
            assert orc.rel_l2(y[b][fine[b]].astype(np.float64), o[b][fine[b]]) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 12, 16, 40])
@pytest.mark.parametrize("what", ["one value", "one position", "one dimension", "growing", "falling", "tiny", "keys", "zeros"])
def test_attn_tree_value_range(what, N, positions):
    """Caches whose values (or keys) span many binary orders, in every
    direction: outputs within the layer tolerance of the definition, dimension
    by dimension of W_O's input (W_O = identity here)."""
    B, nh, nkv, hd, S = 2, 8, 2, 16, 150
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 128, nh, nkv, hd, S, [120, 77], 97, "tree", positions)
    w["wo"] = np.eye(128, dtype=np.float32)
    x *= np.float32(1e-30) if what == "tiny" else 1
    ramp = np.float32(2.0) ** np.linspace(-30, 30, S, dtype=np.float32)[None, :, None]
    kc_all, vc_all = kc, vc
    kc, vc = kc[:, :S], vc[:, :S]            # (the rows that a sequence reaches)
    if what == "one value":
        vc[:, 40, 5] = 1e9
    elif what == "one position":
        vc[:, 70] *= np.float32(1e7)
        kc[:, 70] *= 4
    elif what == "one dimension":
        vc[:, :, 3] *= np.float32(1e8)
        vc[:, :, 4] *= np.float32(1e-8)
    elif what == "growing":
        vc *= ramp
    elif what == "falling":
        vc *= ramp[:, ::-1]
    elif what == "tiny":
        vc *= np.float32(1e-30)
        w["wv"] *= 0
    elif what == "keys":
        kc[:, :, 7] *= np.float32(1e5)
        w["wq"][:, 6::16] = w["wq"][:, 7::16] = 0.0
    else:
        vc[:, 16:90] = 0.0
        kc[:, 100:110] = 0.0
    print(f"[gpu-test] value range {what} N={N}", flush=True)
    got = run_tree(x, w, kc_all, vc_all, pos, c, s, par, nh, nkv, hd)
    y, k, v, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par, pos,
                              kc_all, vc_all, nh, nkv, hd)
    assert live.all()
    for j in range(128):
        # the sum's own scale: what it adds, each term's probability near 1 at worst
        ref = y[..., j]
        assert np.abs(got[0][..., j] - ref).max() <= 2e-5 * np.abs(ref).max(), (j, np.abs(got[0][..., j] - ref).max() / np.abs(ref).max())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(27, 60, 100, 6, 3, 24, 50), (400, 4, 64, 4, 2, 16, 30), (13, 50, 260, 5, 1, 40, 20),
                                   (100, 48, 260, 2, 1, 64, 20), (150, 32, 132, 2, 2, 56, 16), (50, 40, 700, 8, 2, 24, 30)],
                         ids=lambda s: "_".join(map(str, s)))
def test_attn_tree_many_rows(shape):
    """Hundreds and thousands of rows: the projections on the matrix cores in
    each of their tiles, widths that no tile divides."""
    B, N, d, nh, nkv, hd, S = shape
    print(f"[gpu-test] tree rows {shape}", flush=True)
    pos = np.random.default_rng(3).integers(0, S, B)
    kind = "holes" if B * N < 2000 else "tree"
    _, live = check_tree(*tree_case(B, N, d, nh, nkv, hd, S, pos, 91, kind), nh, nkv, hd)
    assert live.sum() > B


@pytest.mark.gpu
@pytest.mark.parametrize("N", [8, 16])
def test_attn_tree_number_range(N):
    """Rows and weights at the ends of the float range, among ordinary ones:
    keys and values within 1e-5 of the definition's, row by row."""
    B, nh, nkv, hd, S = 10, 4, 2, 16, 40
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 64, nh, nkv, hd, S, [5] * B, 95, "chain")
    par[:] = -1                              # (every row for itself)
    for i, f in enumerate((1e-30, 1e-36, 1e18, 1e-18, 1.0)):
        x[i] *= np.float32(f)
    x[5, :, 0] = 3e18                        # (its square overflows: the row's 1/rms is 0)
    w["wv"][:, 3] *= np.float32(1e-36)
    w["wv"][:, 4] *= np.float32(1e30)
    w["wv"][:, 5] = 0.0
    print("[gpu-test] tree number range", flush=True)
    y, k, v = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd)
    z = x.astype(np.float64)
    inv = 1.0 / np.sqrt((z ** 2).mean(2, keepdims=True) + np.float64(np.float32(EPS)))
    want = (z * inv * w["rms"].astype(np.float64)) @ w["wv"].astype(np.float64)
    for b in [0, 1, 3, 4, 6, 7, 8, 9]:
        for j in range(nkv * hd):
            ref = want[b, :, j]
            # (sums near the smallest floats keep few bits)
            if np.abs(ref).max() > 1e-33:
                assert np.abs(v[b, :, j] - ref).max() <= 1e-5 * np.abs(want[b][:, j]).max() + 1e-36, (b, j)
    assert np.array_equal(v[:, :, 5], np.zeros((B, N), np.float32))


@pytest.mark.gpu
def test_attn_tree_positions_and_empty_trees():
    """Positions outside the cache, nodes past its end, trees without a
    token, and y in place."""
    x, w, kc, vc, pos, c, s, par = tree_case(6, 9, 128, 8, 2, 16, 32, [-1, 32, 31, 28, 5, 2147483647],
                                             21, "chain")
    par[4] = -2
    print("[gpu-test] tree positions", flush=True)
    _, live = check_tree(x, w, kc, vc, pos, c, s, par, 8, 2, 16)
    assert live.sum(1).tolist() == [0, 0, 1, 4, 0, 0]
    check_tree(x, w, kc, vc, pos, c, s, par, 8, 2, 16, in_place=True)
    check_tree(x, w, kc, vc, pos, c, s, make_parents("none", 6, 9, 1), 8, 2, 16)


@pytest.mark.gpu
def test_attn_tree_nonfinite(positions):
    """NaN in draft buffers, in cache rows at and past pos, and in the rows of
    nodes that are no token reaches nothing; a NaN or infinite token reaches
    itself and its descendants only."""
    B, N, nh, nkv, hd, S = 3, 24, 8, 2, 32, 80
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 128, nh, nkv, hd, S, [0, 37, 55], 31, "tree", positions)
    for b in range(B):
        kc[b, pos[b]:] = np.nan
        vc[b, pos[b]:] = np.inf
    par[1, 5] = -2
    x[1, 5] = np.nan
    print("[gpu-test] tree nonfinite: masked", flush=True)
    clean, live = check_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, fill=np.nan)
    for bad in (np.nan, np.inf):
        x2 = x.copy()
        x2[2, 3, 7] = bad
        hit = np.zeros((B, N), bool)
        hit[2] = [ch is not None and 3 in ch for ch in to.chains(par[2])]
        assert 1 < hit.sum() < N
        y, k, v = run_tree(x2, w, kc, vc, pos, c, s, par, nh, nkv, hd, fill=np.nan)
        assert not np.isfinite(y[hit]).all(1).any()
        ok = live & ~hit
        # (the sequence takes its range with float products: two forms of the
        # same sums, each within the layer tolerance)
        assert orc.rel_l2(y[ok], clean[0][ok]) <= 1e-5 and np.abs(y[ok] - clean[0][ok]).max() <= 1e-4
        assert np.array_equal(y[:2][ok[:2]], clean[0][:2][ok[:2]])
    # An infinite value in the cache reaches its sequence only.
    vc2 = vc.copy()
    vc2[1, 3, 2] = np.inf
    y, _, _ = run_tree(x, w, kc, vc2, pos, c, s, par, nh, nkv, hd)
    assert not np.isfinite(y[1][live[1]]).all(1).any()
    assert np.array_equal(y[[0, 2]][live[[0, 2]]], clean[0][[0, 2]][live[[0, 2]]])


@pytest.mark.gpu
def test_attn_tree_large_scores(positions):
    """Scores of some hundreds: one-hot softmaxes whose maximum moves many
    times; the maximum may come first or last."""
    x, w, kc, vc, pos, c, s, par = tree_case(2, 16, 128, 4, 2, 32, 300, [290, 290], 41, "tree", positions)
    ramp = np.linspace(0.1, 8.0, 300, dtype=np.float32)[:, None]
    kc[0, :300] *= ramp
    kc[1, :300] *= ramp[::-1]
    w["wq"] *= 4
    # (scores to ~400: their fp32 rounding, 2^-24 of 400 twice, moves an
    # exponential by 5e-5; outputs of two near rows follow)
    got = run_tree(x, w, kc, vc, pos, c, s, par, 4, 2, 32)
    y, _, _, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par, pos,
                              kc, vc, 4, 2, 32)
    assert live.all() and orc.rel_l2(got[0], y) <= 5e-5


@pytest.mark.gpu
def test_attn_tree_single_token_is_decode():
    """N = 1 is the decode step: same rows within the layer tolerance, and
    the commit of node 0 makes the same cache."""
    B, S, nh, nkv, hd = 9, 150, 8, 2, 64
    x, w, kc, vc, pos, c, s, par = tree_case(B, 1, 512, nh, nkv, hd, S, np.arange(B) * 17, 51, "chain")
    at = mh.Attn(512, nh, nkv, hd, S)
    at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
    at.set_rope(c, s)
    try:
        y, k, v = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
        dx, dk, dv, dp = dev(x[:, 0]), dev(kc), dev(vc), dev(pos)
        at.decode_dev(dx.ptr, B, dp.ptr, dk.ptr, dv.ptr, EPS)
        assert orc.rel_l2(y[:, 0], dx.to_host()) <= 1e-5
        ko, vo, po = to.commit(k, v, kc, vc, pos, np.zeros((B, 1), np.int32), np.zeros(B, np.int32))
        assert orc.rel_l2(ko, dk.to_host()) <= 1e-6 and orc.rel_l2(vo, dv.to_host()) <= 1e-6
        assert np.array_equal(po, pos + 1)
    finally:
        at.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 8, 512, 8, 2, 64, 900), (40, 12, 256, 8, 2, 32, 200)])
def test_attn_tree_repeats_and_graph(shape, positions):
    """The same bits on a repeat, after a call of another shape, and from each
    replay of a captured graph with eager work between the replays."""
    B, N, d, nh, nkv, hd, S = shape
    pos = np.random.default_rng(6).integers(0, S - N, B)
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, pos, 61, "tree", positions)
    at = mh.Attn(d, nh, nkv, hd, kc.shape[1])
    at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
    at.set_rope(c, s)
    try:
        first = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
        run_tree(x[:, :1].copy(), w, kc, vc, pos, c, s, par[:, :1], nh, nkv, hd, at=at)
        again = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
        for u, v in zip(first, again):
            assert np.array_equal(u, v)
        dx, dk, dv, dpar, dpos = dev(x), dev(kc), dev(vc), dev(par), dev(pos)
        dy, gk, gv = mh.DeviceArray(x.shape), mh.DeviceArray((B, N, nkv * hd)), mh.DeviceArray((B, N, nkv * hd))
        with mh.Graph() as g:
            at.tree_dev(dx.ptr, dy.ptr, B, N, dpar.ptr, dpos.ptr, dk.ptr, dv.ptr, gk.ptr, gv.ptr, EPS)
        try:
            for _ in range(4):
                dy.zero(), gk.zero(), gv.zero()
                g.launch()
                mh.synchronize()
                for u, v in zip(first, (dy, gk, gv)):
                    assert np.array_equal(u, v.to_host())
                small = run_tree(x[:1], w, kc[:1], vc[:1], pos[:1], c, s, par[:1], nh, nkv, hd, at=at)
                assert orc.rel_l2(small[0], first[0][:1]) <= 1e-5
        finally:
            g.close()
    finally:
        at.close()


@pytest.mark.gpu
def test_attn_tree_refusals():
    at = mh.Attn(64, 4, 2, 16, 32)
    try:
        L, P = mh.lib(), C.c_void_p
        a = mh.DeviceArray((1 << 16,))
        base = a.ptr.value
        x, y, kc, vc, kd, vd, i = (base + 32768 * j for j in range(7))

        def call(x=x, y=y, B=1, N=4, par=i, pos=i, kc=kc, vc=vc, kd=kd, vd=vd):
            return L.moe_hip_attn_tree_dev(at.h, P(x), P(y), B, N, P(par), P(pos), P(kc), P(vc), P(kd),
                                           P(vd), EPS, None)

        assert call(B=0) == 0
        assert call(B=-1) == 1 and call(N=0) == 1 and call(N=65) == 1
        assert call(B=(1 << 20) + 1, N=1) == 2
        for name in ("x", "y", "par", "pos", "kc", "vc", "kd", "vd"):
            assert call(**{name: None}) == 1, name
        for name in ("x", "y", "kc", "vc", "kd", "vd"):
            assert call(**{name: locals()[name] + 4}) == 1, name       # alignment
        wide = mh.Attn(64, 32, 32, 8, 4)     # (addresses that are never read)
        far = [P((j + 1) << 40) for j in range(8)]
        assert L.moe_hip_attn_tree_dev(wide.h, far[0], far[1], 1 << 19, 1, *far[2:8], EPS, None) == 2
        wide.close()
        assert call(y=kc) == 1 and call(y=vc + 16) == 1 and call(y=i) == 1 and call(kd=i) == 1
        assert call(y=x + 64) == 1 and call(kd=vd) == 1 and call(kd=x) == 1 and call(vd=kc) == 1
        layer = mh.Layer(128, 64, 2, 1)
        assert L.moe_hip_tree_block_dev(at.h, layer.h, P(x), P(x), 1, 4, P(i), P(i), P(kc), P(vc),
                                        P(kd), P(vd), EPS, None, None, None) == 1    # widths differ
        layer.close()
    finally:
        at.close()


# ---------------------------------------------------------------- verification
def verify_case(B, N, V, kind, seed, probs=True, sharp=2.0):
    rng = np.random.default_rng(seed)
    soft = lambda z: (np.exp(z - z.max(-1, keepdims=True)) / np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731,E501
    z = sharp * rng.standard_normal((B, N, V))
    p, q = soft(z), soft(0.7 * z + 0.5 * sharp * rng.standard_normal((B, N, V)))
    par = make_parents(kind, B, N, seed)
    tok = np.zeros((B, N), np.int32)
    for b in range(B):
        for i in range(N):
            r = q[b, par[b, i]] if 0 <= par[b, i] < i else q[b, 0]
            tok[b, i] = rng.choice(V, p=r / r.sum(dtype=np.float64).astype(np.float64)) if V > 1 else 0
    return p, q if probs else None, par, tok, rng.random((B, N)).astype(np.float32), rng.random(B).astype(np.float32)


def run_verify(p, q, par, tok, ua, us, pad=0, stream=None):
    B, N, V = p.shape
    wide = lambda t: dev(np.concatenate((t, np.full((B, N, pad), np.nan, np.float32)), 2)) if pad else dev(t)  # noqa: E731,E501
    dp, dq = wide(p), wide(q) if q is not None else None
    dpar, dtok, dua, dus = dev(par), dev(tok), dev(ua), dev(us)
    out = [mh.DeviceArray.from_host(np.full(sh, 77, np.int32)) for sh in ((B, N), (B,), (B,))]
    mh.tree_verify_dev(dp.ptr, V + pad, dq.ptr if dq else None, V + pad, B, N, V, dpar.ptr, dtok.ptr,
                       dua.ptr, dus.ptr, *[o.ptr for o in out], stream)
    return [o.to_host() for o in out]


def check_verify(*case, pad=0):
    got, want = run_verify(*case, pad=pad), to.verify(*case)
    for name, g, o in zip(("path", "n_acc", "next"), got, want):
        assert np.array_equal(g, o), (name, np.argwhere(g != o)[:5], g, o)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [True, False], ids=["drawn", "looked-up"])
@pytest.mark.parametrize("kind", ["chain", "tree", "star", "forest", "holes", "ragged"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 1, 130), (3, 2, 2), (40, 6, 7), (30, 17, 64),
                                   (20, 64, 1000), (7, 9, 4096), (3, 5, 50001)],
                         ids=lambda s: "_".join(map(str, s)))
def test_tree_verify(shape, kind, probs):
    print(f"[gpu-test] verify {shape} {kind} {probs}", flush=True)
    case = verify_case(*shape, kind, 5 + shape[1], probs)
    path, n_acc, _ = check_verify(*case)
    if shape == (20, 64, 1000) and kind == "tree" and probs:     # (paths of several lengths)
        assert len(set(n_acc.tolist())) > 2
    check_verify(*case, pad=3)


@pytest.mark.gpu
def test_tree_verify_edges():
    """Equal distributions (nothing left after a rejection), one-hot targets
    (greedy), zeros, u at both ends, tokens outside the vocabulary, NaN,
    infinite and negative entries, sequences without a root."""
    print("[gpu-test] verify edges", flush=True)
    p, q, par, tok, ua, us = verify_case(24, 12, 300, "tree", 71)
    check_verify(p, p.copy(), par, tok, ua, us)
    check_verify(p, p.copy(), par, tok, np.ones_like(ua), us)      # (u = 1: p = q is rejected, nothing left)
    hot = np.zeros_like(p)
    hot[np.arange(24)[:, None], np.arange(12), p.argmax(2)] = 1.0
    tok2 = tok.copy()
    for b in range(0, 24, 2):
        for i in range(1, 12):
            tok2[b, i] = p[b, par[b, i]].argmax()
    for t in (tok, tok2):
        path, n_acc, nxt = check_verify(hot, q, par, t, ua, us)
        check_verify(hot, None, par, t, ua, us)
        last = path[np.arange(24), n_acc]
        assert np.array_equal(nxt, p.argmax(2)[np.arange(24), last])
    for u in (0.0, np.float32(1.0 - 2.0 ** -24)):
        check_verify(p, q, par, tok, np.full_like(ua, u), np.full_like(us, u))
        check_verify(p, None, par, tok, np.full_like(ua, u), np.full_like(us, u))
    t3 = tok.copy()
    t3[:, 1::3] = -1
    t3[:, 2::3] = 300
    t3[:, 3::5] = 2147483647
    check_verify(p, q, par, t3, ua, us)
    check_verify(p, None, par, t3, ua, us)
    q0 = q.copy()
    q0[:, :, ::2] = 0.0
    check_verify(p, q0, par, tok, ua, us)
    check_verify(np.zeros_like(p), q, par, tok, ua, us)
    bad = p.copy()
    bad[::3, :, 5] = np.nan
    bad[1::3, :, 9] = -0.25
    bad[2::3, :, 11] = np.inf
    for qq in (q, None):
        check_verify(bad, qq, par, tok, ua, us)
    par2 = par.copy()
    par2[::2, 0] = [-2, 0, 5, 12, -2, 1, 1, -7, 3, 64, 9, -3]
    path, n_acc, nxt = check_verify(p, q, par2, tok, ua, us)
    assert (n_acc[::2] == -1).all() and (nxt[::2] == -1).all() and (path[::2] == -1).all()
    # rows of q that no child was drawn from are not read
    q2 = q.copy()
    for b in range(24):
        for i in range(12):
            if i not in par[b]:
                q2[b, i] = np.nan
    assert np.isnan(q2).any()
    got = check_verify(p, q2, par, tok, ua, us)
    for u, v in zip(got, check_verify(p, q, par, tok, ua, us)):
        assert np.array_equal(u, v)
    # every child the same token
    check_verify(p, q, par, np.full_like(tok, 17), ua, us)
    check_verify(p, None, make_parents("star", 24, 12, 0), np.full_like(tok, 17), ua, us)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "tree", "ragged"])
def test_tree_verify_likely_drafts(kind):
    """Looked-up drafts that are often the target's likeliest token (p of 0.5
    and more): accepted paths of many lengths."""
    B, N, V = 40, 24, 700
    p, _, par, tok, ua, us = verify_case(B, N, V, kind, 72, False, sharp=3.0)
    for b in range(B):
        for i in range(1, N):
            if 0 <= par[b, i] < i and (b + i) % 4:
                tok[b, i] = p[b, par[b, i]].argsort()[-1 - i % 3]
    _, n_acc, _ = check_verify(p, None, par, tok, ua, us)
    assert len(set(n_acc.tolist())) > 2


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [False, True], ids=["peaked", "flat-target"])
@pytest.mark.parametrize("kind", ["star", "tree"])
@pytest.mark.parametrize("shape", [(2, 30, 20000), (1, 40, 70001), (9, 12, 9000)], ids=lambda s: "_".join(map(str, s)))
def test_tree_verify_many_rejections(shape, kind, flat):
    """Large vocabularies (several workgroups per sequence) and many rejected
    children at a node: later passes read what an earlier one left; a flat
    target against a peaked draft leaves nearly every token."""
    B, N, V = shape
    print(f"[gpu-test] verify rejections {shape} {kind} {flat}", flush=True)
    rng = np.random.default_rng(N + V)
    soft = lambda z: (np.exp(z - z.max(-1, keepdims=True)) / np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731,E501
    z = rng.standard_normal((B, N, V))
    p, q = soft(0.1 * z if flat else 2 * z), soft(3 * rng.standard_normal((B, N, V)))
    par = make_parents(kind, B, N, 1)
    up = np.maximum(par, 0)
    tok = (np.log(q[np.arange(B)[:, None], up]) + rng.gumbel(size=(B, N, V))).argmax(2).astype(np.int32)
    us = rng.random(B).astype(np.float32)
    for ua in (rng.random((B, N)), 0.5 + 0.5 * rng.random((B, N)), np.ones((B, N))):
        _, n_acc, _ = check_verify(p, q, par, tok, ua.astype(np.float32), us)
        check_verify(p, None, par, tok, ua.astype(np.float32), us)


@pytest.mark.gpu
def test_tree_verify_repeats_and_graph():
    """The same results from each replay of a captured call, between eager
    calls of other shapes (the arrival counters are back at zero)."""
    cases = [verify_case(3, 9, 30011, "tree", 7), verify_case(40, 6, 9000, "tree", 8),
             verify_case(1, 12, 50000, "star", 9)]
    first = [run_verify(*c) for c in cases]
    p, q, par, tok, ua, us = cases[0]
    B, N, V = p.shape
    d = [dev(t) for t in (p, q, par, tok, ua, us)]
    out = [mh.DeviceArray(sh, np.int32) for sh in ((B, N), (B,), (B,))]
    with mh.Graph() as g:
        mh.tree_verify_dev(d[0].ptr, V, d[1].ptr, V, B, N, V, *[t.ptr for t in d[2:] + out])
    try:
        for k in range(4):
            for o in out:
                o.zero()
            g.launch()
            mh.synchronize()
            for o, w in zip(out, first[0]):
                assert np.array_equal(o.to_host(), w)
            for u, v in zip(run_verify(*cases[1 + k % 2]), first[1 + k % 2]):
                assert np.array_equal(u, v)
    finally:
        g.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 5, 600001), (3, 1, 65600), (5, 16, 65537), (40, 6, 66000), (64, 4, 64513), (65, 4, 64513)],
                         ids=lambda s: "_".join(map(str, s)))
def test_tree_verify_long_rows(shape):
    """Rows long enough that a sequence's workgroups share every pass, with
    rejections before and after accepted nodes; replayed from a graph between
    eager calls of another shape, with the same results each time."""
    B, N, V = shape
    print(f"[gpu-test] verify long rows {shape}", flush=True)
    rng = np.random.default_rng(N + V)

    def dist(scale):   # (a few likely tokens over a flat rest)
        z = scale * rng.random((B, N, V), dtype=np.float32) ** 8
        z /= z.sum(-1, keepdims=True, dtype=np.float64)
        return z.astype(np.float32)

    p = dist(1.0)
    q = 0.5 * (p + np.roll(p, 1, axis=-1))
    par = make_parents("tree", B, N, 3)
    up = np.maximum(par, 0)
    pick = np.empty((B, N), np.int32)
    for b in range(B):
        for i in range(N):
            pick[b, i] = np.searchsorted(np.cumsum(q[b, up[b, i]], dtype=np.float64), rng.random() * 0.999)
    us = rng.random(B).astype(np.float32)
    for ua in (rng.random((B, N)), 0.6 + 0.4 * rng.random((B, N))):
        ua = ua.astype(np.float32)
        want = check_verify(p, q, par, pick, ua, us)
    check_verify(p, None, par, pick, ua, us)
    if B > 1:                                # no root, nothing to draw from, no number
        par2, p2 = par.copy(), p.copy()
        par2[0, 0] = -2
        p2[1] = 0.0
        p2[2, :, V // 2] = np.nan
        p2[B - 1, :, 9] = np.inf
        check_verify(p2, q, par2, pick, ua, us)
    other = verify_case(3, 9, 30011, "tree", 7)
    first = run_verify(*other)
    d = [dev(t) for t in (p, q, par, pick, ua, us)]
    out = [mh.DeviceArray(sh, np.int32) for sh in ((B, N), (B,), (B,))]
    with mh.Graph() as g:
        mh.tree_verify_dev(d[0].ptr, V, d[1].ptr, V, B, N, V, *[t.ptr for t in d[2:] + out])
    try:
        for _ in range(3):
            for o in out:
                o.zero()
            g.launch()
            mh.synchronize()
            for o, w in zip(out, want):
                assert np.array_equal(o.to_host(), w)
            for u, v in zip(run_verify(*other), first):
                assert np.array_equal(u, v)
    finally:
        g.close()


@pytest.mark.gpu
def test_tree_verify_all_tokens_tried():
    """Looked-up drafts that cover the whole vocabulary, every one rejected
    but the last possible: the walk ends with the target's own row or an
    accepted token."""
    V, N = 16, 40
    rng = np.random.default_rng(3)
    p = rng.dirichlet(np.ones(V), (6, N)).astype(np.float32)
    par = make_parents("star", 6, N, 0)
    tok = np.tile(np.arange(N) % V, (6, 1)).astype(np.int32)
    one = np.ones((6, N), np.float32)
    check_verify(p, None, par, tok, one, rng.random(6).astype(np.float32))
    check_verify(p, None, par, tok, one * 2, rng.random(6).astype(np.float32))


# ---------------------------------------------------------------------- commit
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 4), (2, 3, 8, 20, 16), (40, 5, 16, 60, 128),
                                   (3, 7, 64, 70, 20), (2, 2, 4, 9, 1024)],
                         ids=lambda s: "_".join(map(str, s)))
@pytest.mark.parametrize("where", ["apart", "in-place", "none"])
def test_tree_commit(shape, where):
    """(blocks, B, N, max_seq, kv_dim): accepted rows bit for bit, everything
    else untouched; paths with entries outside the tree, counts beyond it,
    positions outside the cache."""
    L, B, N, S, kd = shape
    print(f"[gpu-test] commit {shape} {where}", flush=True)
    rng = np.random.default_rng(L + N)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    kds, vds, kcs, vcs = ([f(B, n, kd) for _ in range(L)] for n in (N, N, S, S))
    pos = rng.integers(0, S, B).astype(np.int32)
    n_acc = rng.integers(0, N, B).astype(np.int32)
    path = np.full((B, N), -1, np.int32)
    for b in range(B):
        path[b, :n_acc[b] + 1] = np.sort(rng.permutation(N)[:n_acc[b] + 1])
    if B > 4:
        pos[0], pos[1], n_acc[2], n_acc[3], path[4, 0] = -1, S, -1, 2 * N, N
    d = [[dev(a) for a in v] for v in (kds, vds, kcs, vcs)]
    dpos, dpath, dn = dev(pos), dev(path), dev(n_acc)
    out = {"apart": dev(np.full(B, 55, np.int32)), "in-place": dpos, "none": None}[where]
    mh.tree_commit_dev(*[[a.ptr for a in v] for v in d], B, N, kd, S, dpos.ptr, dpath.ptr, dn.ptr,
                       out.ptr if out else None)
    for l in range(L):
        ko, vo, po = to.commit(kds[l], vds[l], kcs[l], vcs[l], pos, path, n_acc)
        assert np.array_equal(d[2][l].to_host(), ko) and np.array_equal(d[3][l].to_host(), vo), l
        assert np.array_equal(d[0][l].to_host(), kds[l])
    assert np.array_equal(dpos.to_host(), po if where == "in-place" else pos)
    if where == "apart":
        assert np.array_equal(out.to_host(), po)


# ------------------------------------------------------------------ as a model
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_drafted_steps_equal_decode_steps(kind):
    """Two blocks of attention and MoE: a tree of drafts through
    moe_hip_tree_block_dev, verified and committed, three steps long, against
    the accepted tokens fed one by one through moe_hip_decode_block_dev: the
    caches and the accepted nodes' rows agree."""
    from conftest import CONFIGS
    c4 = CONFIGS["c4"]
    d, F, E, k, nh, nkv, hd, S, V = 128, 256, 4, 2, 8, 2, 16, 60, 50
    B, N, blocks = 5, 9, 2
    rng = np.random.default_rng(81)
    emb = rng.standard_normal((V, d)).astype(np.float32)
    head = rng.standard_normal((d, V)).astype(np.float32) * 0.1
    soft = lambda z: (np.exp(z - z.max(-1, keepdims=True)) / np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731,E501
    ats, layers, rms, tree, step = [], [], [], [], []
    try:
        for l in range(blocks):
            _, w, kc, vc, _, cs, sn = make_case(B, S, [0] * B, 90 + l, d, nh, nkv, hd)
            at = mh.Attn(d, nh, nkv, hd, S)
            at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
            at.set_rope(cs, sn)
            layer = mh.Layer(d, F, E, k)
            layer.fill_synthetic(20 + l, c4["std_router"], c4["std_expert"])
            ats.append(at), layers.append(layer)
            rms.append(dev((1.0 + 0.1 * rng.standard_normal(d)).astype(np.float32)))
            tree.append((dev(kc), dev(vc))), step.append((dev(kc), dev(vc)))
        pos = np.array([0, 3, 16, 31, 20], np.int32)
        dpos = dev(pos)
        root = rng.integers(0, V, B).astype(np.int32)
        drafts = [(mh.DeviceArray((B, N, nkv * hd)), mh.DeviceArray((B, N, nkv * hd))) for _ in range(blocks)]
        total = 0
        for it in range(3):
            par = make_parents(kind, B, N, it)
            q = np.tile(soft(rng.standard_normal((B, 1, V))), (1, N, 1))
            tok = np.array([rng.choice(V, N, p=r[0].astype(np.float64) / r[0].astype(np.float64).sum()) for r in q], np.int32)
            tok[:, 0] = root
            dx, dpar = dev(emb[tok]), dev(par)
            for l in range(blocks):
                ats[l].tree_block_dev(layers[l], rms[l].ptr, dx.ptr, B, N, dpar.ptr, dpos.ptr,
                                      tree[l][0].ptr, tree[l][1].ptr, drafts[l][0].ptr, drafts[l][1].ptr, EPS)
            rows = dx.to_host()
            p = soft(0.2 * rows @ head)
            ua, us = rng.random((B, N)).astype(np.float32), rng.random(B).astype(np.float32)
            path, n_acc, nxt = check_verify(p, q, par, tok, ua, us)
            dpath, dn = dev(path), dev(n_acc)
            mh.tree_commit_dev(*[[t.ptr for t in v] for v in zip(*[(*a, *b) for a, b in zip(drafts, tree)])],
                               B, N, nkv * hd, S, dpos.ptr, dpath.ptr, dn.ptr, dpos.ptr)
            # the same tokens one by one
            for j in range(int(n_acc.max()) + 1):
                on = n_acc >= j
                node = np.where(on, path[:, j], 0)
                at_pos = dev(np.where(on, pos + j, -1).astype(np.int32))     # (others sit out)
                sx = dev(emb[tok[np.arange(B), node]])
                for l in range(blocks):
                    ats[l].decode_block_dev(layers[l], rms[l].ptr, sx.ptr, B, at_pos.ptr, step[l][0].ptr,
                                            step[l][1].ptr, EPS)
                got = sx.to_host()
                assert orc.rel_l2(rows[np.arange(B), node][on], got[on]) <= 1e-5
            pos = pos + n_acc + 1
            total += int(n_acc.sum())
            assert np.array_equal(dpos.to_host(), pos)
            for (a, b), (e, f) in zip(tree, step):
                for u, v in ((a, e), (b, f)):
                    u, v = u.to_host(), v.to_host()
                    for b_ in range(B):
                        assert orc.rel_l2(u[b_, :pos[b_]], v[b_, :pos[b_]]) <= 1e-5
                        assert np.array_equal(u[b_, pos[b_]:], v[b_, pos[b_]:])
            root = nxt
        assert total > 3      # (drafts were accepted)
    finally:
        for a in ats + layers:
            a.close()


def step_case(seed, B, N, S, V, d, nh, nkv, hd):
    """One block's attention with its caches, and a step's p, q, tokens and
    random numbers."""
    rng = np.random.default_rng(seed)
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, rng.integers(0, 20, B), seed, "tree")
    at = mh.Attn(d, nh, nkv, hd, S)
    at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
    at.set_rope(c, s)
    p, q, _, tok, ua, us = verify_case(B, N, V, "tree", seed)
    return at, [dev(a) for a in (x, kc, vc, np.asarray(pos, np.int32), par, p, q, tok, ua, us)]


def run_step(at, t, out, B, N, S, V, kd, stream=None):
    """Attention, verification and the commit (positions in place)."""
    x, kc, vc, pos, par, p, q, tok, ua, us = t
    y, kdr, vdr, path, n_acc, nxt = out
    at.tree_dev(x.ptr, y.ptr, B, N, par.ptr, pos.ptr, kc.ptr, vc.ptr, kdr.ptr, vdr.ptr, EPS, stream)
    mh.tree_verify_dev(p.ptr, V, q.ptr, V, B, N, V, par.ptr, tok.ptr, ua.ptr, us.ptr, path.ptr,
                       n_acc.ptr, nxt.ptr, stream)
    mh.tree_commit_dev([kdr.ptr], [vdr.ptr], [kc.ptr], [vc.ptr], B, N, kd, S, pos.ptr, path.ptr,
                       n_acc.ptr, pos.ptr, stream)


def step_outputs(B, N, d, kd):
    return [mh.DeviceArray((B, N, d)), mh.DeviceArray((B, N, kd)), mh.DeviceArray((B, N, kd)),
            mh.DeviceArray((B, N), np.int32), mh.DeviceArray((B,), np.int32), mh.DeviceArray((B,), np.int32)]


STEP = (6, 7, 90, 70000, 128, 8, 2, 16)   # B, N, S, V, d, nh, nkv, hd


@pytest.mark.gpu
def test_captured_steps_equal_eager_steps():
    """A whole step as a graph, replayed while the positions move on, another
    graph of another shape (the same workspaces) and eager calls between the
    replays: caches, positions and results as from eager steps, bit for bit."""
    print("[gpu-test] captured steps", flush=True)
    B, N, S, V, d, nh, nkv, hd = STEP
    kd = nkv * hd
    at, t = step_case(5, *STEP)
    at2, t2 = step_case(5, *STEP)
    other = (40, 4, 60, 9000, 64, 4, 2, 16)
    at3, t3 = step_case(6, *other)
    graphs = []
    try:
        out, out2, out3 = step_outputs(B, N, d, kd), step_outputs(B, N, d, kd), step_outputs(40, 4, 64, 32)
        small = (other[0], other[1], other[2], other[3], 32)
        run_step(at3, t3, out3, *small)                       # (the workspace at its size)
        run_step(at2, t2, out2, B, N, S, V, kd)
        first = [a.to_host() for a in out2]
        with mh.Graph() as g:
            run_step(at, t, out, B, N, S, V, kd)
        graphs.append(g)
        with mh.Graph() as g3:
            run_step(at3, t3, out3, *small)
        graphs.append(g3)
        for it in range(4):
            if it:
                run_step(at2, t2, out2, B, N, S, V, kd)
            g3.launch()
            g.launch()
            g3.launch()
            mh.synchronize()
            if it == 0:
                for a, b in zip(out, first):
                    assert np.array_equal(a.to_host(), b)
            for a, b in zip(out + t, out2 + t2):
                assert np.array_equal(a.to_host(), b.to_host()), it
        assert (t[3].to_host() > 20).any()
    finally:
        for g in graphs:
            g.close()
        for a in (at, at2, at3):
            a.close()


@pytest.mark.gpu
def test_steps_on_a_caller_stream():
    """The same steps on a stream of the caller's."""
    print("[gpu-test] steps on a caller stream", flush=True)
    B, N, S, V, d, nh, nkv, hd = STEP
    kd = nkv * hd
    at, t = step_case(5, *STEP)
    at2, t2 = step_case(5, *STEP)
    hip = C.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so"))
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    try:
        out, out2 = step_outputs(B, N, d, kd), step_outputs(B, N, d, kd)
        for _ in range(2):
            run_step(at2, t2, out2, B, N, S, V, kd)
        mh.synchronize()
        for _ in range(2):
            run_step(at, t, out, B, N, S, V, kd, stream)
        assert hip.hipStreamSynchronize(stream) == 0
        for a, b in zip(out + t, out2 + t2):
            assert np.array_equal(a.to_host(), b.to_host())
    finally:
        hip.hipStreamDestroy(stream)
        at.close()
        at2.close()


def part_of(a, start, shape, dtype=np.float32):
    """A host copy of `shape` elements of device array a from element start."""
    out = np.empty(shape, dtype)
    mh.check(mh.lib().moe_hip_memcpy(out.ctypes.data_as(C.c_void_p), C.c_void_p(a.ptr.value + start * out.itemsize),
                                     out.nbytes, 2))
    return out


def put_part(a, start, values):
    v = np.ascontiguousarray(values)
    mh.check(mh.lib().moe_hip_memcpy(C.c_void_p(a.ptr.value + start * v.itemsize), v.ctypes.data_as(C.c_void_p), v.nbytes, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 20])
def test_offsets_past_32_bits(N):
    """Caches of more than 2^31 floats: the last sequence's attention equals
    its attention alone on its own part of them, and its commit lands there."""
    B, S, d, nh, nkv, hd = 300, 60000, 128, 8, 2, 64
    kd = nkv * hd
    print(f"[gpu-test] tree offsets past 32 bits N={N}", flush=True)
    assert (B - 1) * S * kd > 1 << 31
    _, w, _, _, _, _, _ = make_case(1, 4, [0], 5, d, nh, nkv, hd)
    cs, sn = orc.rope_tables(S, hd, 10000.0)
    at = mh.Attn(d, nh, nkv, hd, S)
    at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
    at.set_rope(cs, sn)
    kc, vc = mh.DeviceArray((B, S, kd)), mh.DeviceArray((B, S, kd))
    try:
        for a, seed in ((kc, 1), (vc, 2)):
            mh.fill_normal_dev(a.ptr, B * S * kd, seed, 0, 0.0, 1.0)
        rng = np.random.default_rng(7)
        x = rng.standard_normal((B, N, d)).astype(np.float32)
        pos = np.full(B, 5, np.int32)
        pos[-1] = S - N - 1
        par = make_parents("tree", B, N, 4)
        dx, dpos, dpar = dev(x), dev(pos), dev(par)
        y, kdr, vdr = mh.DeviceArray((B, N, d)), mh.DeviceArray((B, N, kd)), mh.DeviceArray((B, N, kd))
        at.tree_dev(dx.ptr, y.ptr, B, N, dpar.ptr, dpos.ptr, kc.ptr, vc.ptr, kdr.ptr, vdr.ptr, EPS)
        one = [mh.DeviceArray((1, N, n)) for n in (d, kd, kd)]
        off = (B - 1) * S * kd * 4
        last = [dev(a[-1:]) for a in (x, par, pos)]
        at.tree_dev(last[0].ptr, one[0].ptr, 1, N, last[1].ptr, last[2].ptr,
                    C.c_void_p(kc.ptr.value + off), C.c_void_p(vc.ptr.value + off), one[1].ptr, one[2].ptr, EPS)
        for a, b in zip((y, kdr, vdr), one):
            assert orc.rel_l2(a.to_host()[-1], b.to_host()[0]) <= 1e-5
        path = np.full((B, N), -1, np.int32)
        path[:, 0], path[:, 1] = 0, N - 1
        n_acc = np.ones(B, np.int32)
        at0 = (B - 1) * S * kd + int(pos[-1]) * kd
        before = part_of(kc, at0 + 2 * kd, (kd,))
        dpath, dn = dev(path), dev(n_acc)
        mh.tree_commit_dev([kdr.ptr], [vdr.ptr], [kc.ptr], [vc.ptr], B, N, kd, S, dpos.ptr, dpath.ptr, dn.ptr, dpos.ptr)
        k, v = kdr.to_host(), vdr.to_host()
        assert np.array_equal(part_of(kc, at0, (2, kd)), k[-1, [0, N - 1]])
        assert np.array_equal(part_of(vc, at0, (2, kd)), v[-1, [0, N - 1]])
        assert np.array_equal(part_of(kc, at0 + 2 * kd, (kd,)), before)
        assert np.array_equal(dpos.to_host(), pos + 2)
    finally:
        at.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(100, 3, 1000), (30, 10, 70000)], ids=lambda s: "_".join(map(str, s)))
def test_tree_verify_rows_far_apart(shape):
    """Rows 2^24 floats apart, p and q side by side in them: offsets past 32
    bits."""
    B, N, V = shape
    print(f"[gpu-test] verify rows far apart {shape}", flush=True)
    ld = 1 << 24
    p, q, par, tok, ua, us = verify_case(*shape, "tree", 21)
    a = mh.DeviceArray((B * N * ld,))
    for r in range(B * N):
        put_part(a, r * ld, p.reshape(-1, V)[r])
        put_part(a, r * ld + V, q.reshape(-1, V)[r])
    out = [mh.DeviceArray(sh, np.int32) for sh in ((B, N), (B,), (B,))]
    d = [dev(t) for t in (par, tok, ua, us)]
    mh.tree_verify_dev(a.ptr, ld, C.c_void_p(a.ptr.value + 4 * V), ld, B, N, V, *[t.ptr for t in d + out])
    for o, want in zip(out, to.verify(p, q, par, tok, ua, us)):
        assert np.array_equal(o.to_host(), want)


@pytest.mark.gpu
def test_many_sequences():
    """Thousands of sequences: attention as in calls of fifty, verification as
    the oracle's."""
    B, N, d, nh, nkv, hd, S = 4000, 5, 64, 4, 2, 16, 24
    print("[gpu-test] tree many sequences", flush=True)
    pos = np.random.default_rng(3).integers(0, S, B)
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, pos, 33, "tree")
    at = mh.Attn(d, nh, nkv, hd, S)
    at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
    at.set_rope(c, s)
    try:
        whole = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
        for b in range(0, B, 800):
            cut = slice(b, b + 50)
            for g, o in zip(whole, run_tree(x[cut], w, kc[cut], vc[cut], pos[cut], c, s, par[cut], nh, nkv, hd, at=at)):
                assert orc.rel_l2(g[cut], o) <= 1e-5
    finally:
        at.close()
    check_verify(*verify_case(3000, 4, 60, "tree", 34))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 4), (2, 16), (3, 40), (20, 12), (130, 3), (130, 8)], ids=lambda s: "x".join(map(str, s)))
def test_attn_tree_bits_whatever_ran_before(shape, positions):
    """Trees with unused nodes and nodes past the cache's end, after calls that
    leave zero, ordinary, very large and NaN queries in the workspace: the
    same bits each time, in every block size and projection form."""
    B, N = shape
    nh, nkv, hd, d, S = 8, 2, 16, 128, 300
    print(f"[gpu-test] tree after other calls {shape}", flush=True)
    pos = np.resize([S - 2, 200, 17], B)
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, pos, 130 + N, "holes", positions)
    if N > 4:
        par[:, N // 2] = -2
    else:
        par[:, 1] = -2
    total = kc.shape[1]
    dead = [ch is None for b in range(B) for ch in to.chains(par[b])]
    assert any(dead) and not all(dead)
    own = []
    for scale in (1.0, 3000.0):
        own.append(mh.Attn(d, nh, nkv, hd, total))
        own[-1].load((scale * w["wq"]).astype(np.float32), w["wk"], w["wv"], w["wo"], w["rms"])
        own[-1].set_rope(c, s)
    every = np.full((B, N), -1, np.int32)
    try:
        first = None
        for at, before in ((own[0], 0 * x), (own[0], x), (own[1], x), (own[0], np.full_like(x, np.nan))):
            run_tree(before, w, kc, vc, np.zeros(B, np.int32), c, s, every, nh, nkv, hd, at=at)
            got = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=own[0])
            first = first or got
            for u, v in zip(first, got):
                assert np.array_equal(u, v)
    finally:
        for at in own:
            at.close()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 8, 12, 40])
def test_attn_tree_key_outliers(N):
    """One key dimension near the largest that the split form takes, where the
    queries are zero; the other keys small, the queries large: the attention
    is the small ones'.  Scores are sums of 62 products around 1 (log2 units), whose
    operands carry some roundings of 2^-24 each: sqrt(62) 3e-7 ln 2 = 2e-6 of
    an exponential in the root mean square; the layer tolerance, on the rows of
    attention alone."""
    B, nh, nkv, hd, S = 2, 8, 2, 64, 150
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 512, nh, nkv, hd, S, [140, 77], 140 + N, "tree", "many")
    w["wo"] = np.eye(512, dtype=np.float32)
    norm = np.sqrt((w["wq"].astype(np.float64) ** 2).sum(0).mean())
    w["wq"] = (w["wq"] * (333.0 * 8 / 1.4427 / norm)).astype(np.float32)     # queries of 333 in log2 units
    w["wk"] = (w["wk"] * (0.003 / np.sqrt((w["wk"].astype(np.float64) ** 2).sum(0).mean()))).astype(np.float32)
    w["wq"][:, 62::64] = w["wq"][:, 63::64] = 0.0
    kc[:, :S] = np.random.default_rng(N).standard_normal((B, S, nkv * hd)).astype(np.float32) * np.float32(0.003)
    kc[:, :S:8, 62::64] = 4000.0
    vc[:, :S] = np.random.default_rng(N + 1).standard_normal((B, S, nkv * hd)).astype(np.float32)
    print(f"[gpu-test] key outliers N={N}", flush=True)
    got = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd)
    y, _, _, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par, pos, kc, vc, nh, nkv, hd)
    rel = orc.rel_l2((got[0].astype(np.float64) - x)[live], (y - x)[live])
    print(f"[gpu-test]   rel-L2 {rel:.2e}", flush=True)
    assert live.all() and rel <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [22, 27, 32])
@pytest.mark.parametrize("N", [2, 8, 12, 40])
def test_attn_tree_small_values_of_a_likely_position(N, gap):
    """A position that takes nearly all of the attention and has values 1e-5 of
    the others', which are 2^gap less likely: the output is as small as its
    values, and the others' probabilities and values must not blur it.  The
    layer tolerance, on the rows of attention alone (W_O = 1e6, so that x
    does not drown them)."""
    B, nh, nkv, hd, S = 2, 8, 2, 64, 150
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 512, nh, nkv, hd, S, [140, 77], 150 + N, "tree", "many")
    rng = np.random.default_rng(gap)
    w["wo"] = (1e6 * np.eye(512)).astype(np.float32)
    x[:, :, 0] = 10.0
    w["wq"][:, 62::64] = w["wq"][:, 63::64] = 0.0
    w["wq"] *= np.float32(0.02)
    w["wq"][0, 62::64] = 1.0                 # (a pair that RoPE hardly turns)
    kc[:, :S] = rng.standard_normal((B, S, nkv * hd)).astype(np.float32)
    vc[:, :S] = rng.standard_normal((B, S, nkv * hd)).astype(np.float32)
    kc[:, :S, 62::64] = kc[:, :S, 63::64] = 0.0
    w["wk"][:, 62::64] = w["wk"][:, 63::64] = 0.0
    q = 10.0 * w["rms"][0] / np.sqrt((x.astype(np.float64) ** 2).mean())
    kc[:, 7, 62::64] = gap * 8 / 1.4427 / q
    vc[:, 7] *= np.float32(1e-5)
    print(f"[gpu-test] small values N={N} gap {gap}", flush=True)
    got = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd)
    y, _, _, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par, pos, kc, vc, nh, nkv, hd)
    o = (y - x)[live]
    assert live.all() and np.abs(o).max() < 1e3
    rel = orc.rel_l2((got[0].astype(np.float64) - x)[live], o)
    print(f"[gpu-test]   rel-L2 {rel:.2e}", flush=True)
    assert rel <= 1e-5


@pytest.mark.gpu
def test_tree_verify_looked_up_remainders():
    """Looked-up drafts rejected against nearly all of the mass: what is left
    is a sum of the tokens that are left, not a difference of larger sums.
    Probabilities over 2^60, children that cover the whole support, an
    infinite probability among them."""
    print("[gpu-test] verify looked-up remainders", flush=True)
    one = np.float32(1.0) - np.float32(2.0 ** -24)
    star = lambda n: np.array([[-1] + [0] * n], np.int32)  # noqa: E731
    p = np.zeros((1, 4, 4), np.float32)
    p[0, 0] = [one, 1e-20, 2e-20, 0.0]
    tok = np.array([[0, 0, 1, 2]], np.int32)
    ua = np.array([[0, one, 0.9, 0.5]], np.float32)
    path, n_acc, _ = check_verify(p, None, star(3), tok, ua, np.array([0.5], np.float32))
    assert n_acc[0] == 1 and path[0, 1] == 3
    rng = np.random.default_rng(17)
    B = 200
    for N, V, u in ((12, 11, 1.0), (40, 39, 1.0), (40, 200, 1.0), (64, 63, 0.0), (24, 5000, 0.0)):
        p = np.zeros((B, N, V), np.float32)
        p[:, 0] = 2.0 ** -rng.uniform(0, 60, (B, V))
        p[:, 0] /= p[:, 0].sum(1, keepdims=True)
        p[:, 1:] = 1.0 / V
        tok = np.zeros((B, N), np.int32)
        for b in range(B):
            tok[b, 1:] = rng.permutation(V)[:N - 1] if b % 2 else p[b, 0].argsort()[::-1][:N - 1]
        ua = np.full((B, N), u, np.float32) if u else np.maximum(rng.random((B, N)), 0.97).astype(np.float32)
        par = np.repeat(star(N - 1), B, 0)
        _, n_acc, nxt = check_verify(p, None, par, tok, ua, rng.random(B).astype(np.float32))
        assert u < 1 or N <= V or (n_acc == 0).all()
        # (the first child stays likely to be rejected, a later one is infinite)
        p[:, 0, tok[np.arange(B), 3]] = np.inf
        check_verify(p, None, par, tok, ua, rng.random(B).astype(np.float32))


def added_up(r, by_rank=None):
    """A pass's total as the kernel adds it up, bit for bit: segments of 1024
    tokens, of which lane l of a wave holds 256 e + 4 l + i (in this order of e
    and i), the lanes' sums by a tree.  by_rank: the segment's tokens that this
    marks in the lanes' order, every 64th to a lane (not what the kernel does)."""
    def lanes(v):    # v[..., 64]
        v = v.reshape(*v.shape[:-1], 4, 16)
        for s in (1, 2, 4, 8):
            v = v + np.concatenate((np.zeros_like(v[..., :s]), v[..., :-s]), -1)
        v = v[..., 15]
        return (v[..., 0] + v[..., 1]) + (v[..., 2] + v[..., 3])

    V, segs = len(r), -(-len(r) // 1024)
    full = np.zeros(segs * 1024)
    full[:V] = r
    mine = full.reshape(segs, 4, 64, 4).transpose(0, 2, 1, 3).reshape(segs, 64, 16)
    if by_rank is not None:
        mark = np.zeros(segs * 1024, bool)
        mark[:V] = by_rank
        mark = mark.reshape(segs, 4, 64, 4).transpose(0, 2, 1, 3).reshape(segs, 1024)
        packed = np.zeros((segs, 1024))
        for s in range(segs):
            kept = mine[s].reshape(-1)[mark[s]]
            packed[s, :len(kept)] = kept
        mine = packed.reshape(segs, 16, 64).transpose(0, 2, 1)
    t = np.zeros((segs, 64))
    for k in range(16):
        t = t + mine[..., k]
    t = lanes(t)
    c = -(-segs // 64)
    t = np.concatenate((t, np.zeros(64 * c - segs))).reshape(64, c)
    own = np.zeros(64)
    for k in range(c):
        own = own + t[:, k]
    return lanes(own)


def test_sum_orders_differ():
    """The case below is one where the order decides (else it shows nothing)."""
    p, q, par, tok, ua, us, accepted = tie_case()
    p, q = p[0, 0], q[0, 0]
    first = left_over(p, q, 1.0)
    left = left_over(p, q, 1.0 + added_up(first))
    assert added_up(left) != added_up(left, first > 0)
    assert abs(added_up(left) - left.sum()) <= 1e-14 * left.sum()


def left_over(p, q, a):
    """max(p - a q, 0) in 64 bits, rounded once (a fused multiply-add)."""
    from fractions import Fraction
    return np.array([max(float(Fraction(float(x)) - Fraction(float(a)) * Fraction(float(y))), 0.0) for x, y in zip(p, q)])


_TIE = []


def tie_case():
    """One sequence, a root with three children and a row of 65600 tokens: the
    first two are rejected, the third's acceptance hangs on the last bits of the
    sum of what they leave.  Its p and q are so small that they do not count in
    the sums; p / q is a fraction as near to a + u W as 24-bit numbers come."""
    from fractions import Fraction
    if _TIE:
        return _TIE[0]
    V = 65600
    for seed in range(40):
        rng = np.random.default_rng(seed)
        p = rng.random(V, dtype=np.float32) ** 8
        p /= p.sum(dtype=np.float64)
        q = (0.5 * (p + np.roll(p, 1))).astype(np.float32)
        tok = np.array([0, 5, 70, 130], np.int32)
        p[tok[1:3]] = 0.0
        p[tok[3]] = q[tok[3]] = np.float32(2.0 ** -101)
        w1 = added_up(left_over(p, q, 1.0))
        a = 1.0 + w1
        left = left_over(p, q, a)
        rows, ranks = added_up(left), added_up(left, left_over(p, q, 1.0) > 0)
        if rows == ranks:
            continue
        for _ in range(3000):
            u = np.float32(rng.random() * 0.5 + 0.25)
            X = Fraction(a) + Fraction(float(u)) * (Fraction(rows) + Fraction(ranks)) / 2
            h, k, x = (0, 1), (1, 0), X      # convergents h / k of X
            while True:
                n = x.numerator // x.denominator
                h, k = (h[1], n * h[1] + h[0]), (k[1], n * k[1] + k[0])
                if h[1] >= 1 << 24 or k[1] >= 1 << 24:
                    break
                r = float(Fraction(h[1]) - Fraction(a) * k[1])
                yes = [float(u) * k[1] * w < r for w in (rows, ranks)]
                if yes[0] != yes[1] and k[1] >= 1 << 10:
                    p[tok[3]], q[tok[3]] = np.float32(h[1] * 2.0 ** -123), np.float32(k[1] * 2.0 ** -123)
                    N = 4
                    P, Q = np.repeat(p[None, None], N, 1), np.repeat(q[None, None], N, 1)
                    par = np.array([[-1, 0, 0, 0]], np.int32)
                    ua = np.array([[0.0, 0.5, 0.5, u]], np.float32)
                    _TIE.append((P, Q, par, tok[None].copy(), ua, np.array([0.37], np.float32), yes[0]))
                    return _TIE[0]
                if x == n:
                    break
                x = 1 / (x - n)
    raise AssertionError("no such case")


@pytest.mark.gpu
@pytest.mark.parametrize("B", [64, 30, 1])
def test_tree_verify_one_order_of_sums(B):
    """The passes over long rows are shared by a sequence's workgroups, which
    add up a part from a list or, in another's place, from the rows: the same
    order and the same bits by either way, so that equal sequences get equal
    results however the workgroups happen to run."""
    print(f"[gpu-test] verify order of sums B={B}", flush=True)
    p, q, par, tok, ua, us, accepted = tie_case()
    V = p.shape[2]
    d = [dev(np.repeat(t, B, 0)) for t in (par, tok, ua, us)]
    # (all sequences read the same rows: node 0's, and the third child's)
    dp, dq = dev(np.repeat(p, B, 0)), dev(np.repeat(q, B, 0))
    out = [mh.DeviceArray(sh, np.int32) for sh in ((B, 4), (B,), (B,))]
    for _ in range(20):
        mh.tree_verify_dev(dp.ptr, V, dq.ptr, V, B, 4, V, *[t.ptr for t in d + out])
        path, n_acc, nxt = [o.to_host() for o in out]
        assert (n_acc == int(accepted)).all(), n_acc
        assert (path == path[0]).all() and (nxt == nxt[0]).all()


@pytest.mark.gpu
def test_attn_tree_graph_after_new_weights():
    """Weights loaded anew under a captured step: each replay computes with
    the new ones' number range, which the split form of the projections may not
    hold."""
    print("[gpu-test] tree graph after new weights", flush=True)
    B, N, d, nh, nkv, hd, S = 20, 8, 128, 8, 2, 16, 40
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, np.arange(B), 160, "tree")
    x = (x * np.float32(1e14)).astype(np.float32)
    at = mh.Attn(d, nh, nkv, hd, S)
    load = lambda f: at.load(w["wq"], w["wk"], (w["wv"] * np.float32(f)).astype(np.float32), w["wo"], w["rms"])  # noqa: E731
    load(1.0)
    at.set_rope(c, s)
    try:
        run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
        dx, dk, dv, dpar, dpos = dev(x), dev(kc), dev(vc), dev(par), dev(pos)
        dy, gk, gv = mh.DeviceArray(x.shape), mh.DeviceArray((B, N, nkv * hd)), mh.DeviceArray((B, N, nkv * hd))
        with mh.Graph() as g:
            at.tree_dev(dx.ptr, dy.ptr, B, N, dpar.ptr, dpos.ptr, dk.ptr, dv.ptr, gk.ptr, gv.ptr, EPS)
        try:
            xn = x.astype(np.float64)
            xn = xn / np.sqrt((xn ** 2).mean(2, keepdims=True) + EPS) * w["rms"]
            for f in (1.0, 1e-36, 0.0, 1e20, 1.0):
                load(f)
                dy.zero(), gk.zero(), gv.zero()
                g.launch()
                mh.synchronize()
                want = xn @ (w["wv"] * np.float32(f)).astype(np.float64)
                if f:
                    assert orc.rel_l2(gv.to_host() / f, want / f) <= 1e-6, f
                else:
                    assert not gv.to_host().any()
                eager = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=at)
                assert orc.rel_l2(eager[2] / (f or 1), gv.to_host() / (f or 1)) <= 1e-6
        finally:
            g.close()
    finally:
        at.close()


@pytest.mark.gpu
def test_attn_weights_for_many_rows_on_demand():
    """The weights' form for projections of many rows is made by the first call
    that takes it: a program that decodes holds two copies of its weights, not
    three.  A call captured before that has its rows from the other form."""
    print("[gpu-test] attention weights on demand", flush=True)
    hip = C.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so"))

    def free():
        a, b = C.c_size_t(), C.c_size_t()
        assert hip.hipMemGetInfo(C.byref(a), C.byref(b)) == 0
        return a.value

    mh.synchronize()
    d, nh, nkv, hd = 4096, 64, 8, 64
    weights = 4 * (2 * d * nh * hd + 2 * d * nkv * hd)
    before = free()
    at = mh.Attn(d, nh, nkv, hd, 16)
    zero = [np.zeros(s, np.float32) for s in ((d, nh * hd), (d, nkv * hd), (d, nkv * hd), (nh * hd, d))]
    at.load(*zero, np.ones(d, np.float32))
    taken = before - free()
    at.close()
    # (two copies, of which small pieces may lie in memory that the runtime still
    # held; three bf16 terms would be 1.5 times the weights more)
    assert weights < taken < 2.3 * weights, (taken, weights)

    B, N, d, nh, nkv, hd, S = 30, 6, 128, 8, 2, 16, 40
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, d, nh, nkv, hd, S, np.arange(B), 170, "holes")
    ats = [mh.Attn(d, nh, nkv, hd, S) for _ in range(2)]
    for at in ats:
        at.load(w["wq"], w["wk"], w["wv"], w["wo"], w["rms"])
        at.set_rope(c, s)
    try:
        first = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=ats[0], fill=0.0)   # (the workspace)
        dx, dk, dv, dpar, dpos = dev(x), dev(kc), dev(vc), dev(par), dev(pos)
        dy, gk, gv = mh.DeviceArray(x.shape), mh.DeviceArray((B, N, nkv * hd)), mh.DeviceArray((B, N, nkv * hd))
        with mh.Graph() as g:
            ats[1].tree_dev(dx.ptr, dy.ptr, B, N, dpar.ptr, dpos.ptr, dk.ptr, dv.ptr, gk.ptr, gv.ptr, EPS)
        try:
            seen = []
            for it in range(3):
                dy.zero(), gk.zero(), gv.zero()
                g.launch()
                mh.synchronize()
                seen.append([t.to_host() for t in (dy, gk, gv)])
                for u, v, e in zip(seen[0], seen[-1], first):
                    assert np.array_equal(u, v) and orc.rel_l2(v, e) <= 1e-6
                # (an eager call makes the other form, the graph keeps its own)
                for u, v in zip(run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd, at=ats[1], fill=0.0), first):
                    assert np.array_equal(u, v)
        finally:
            g.close()
    finally:
        for at in ats:
            at.close()


@pytest.mark.gpu
def test_block_refused_before_it_changes_rows():
    """A block whose MoE half has more rows than it can index, or would grow
    the workspace under a live graph, is refused with x and the drafts (or
    the caches) as they were."""
    print("[gpu-test] block refusals", flush=True)
    d, F, nh, nkv, hd, S = 64, 8192, 4, 2, 16, 4
    rng = np.random.default_rng(3)
    at, layer = mh.Attn(d, nh, nkv, hd, S), mh.Layer(d, F, 2, 2)
    at.load(*[rng.standard_normal(s).astype(np.float32) for s in ((d, 64), (d, 32), (d, 32), (64, d))], np.ones(d, np.float32))
    at.set_rope(*orc.rope_tables(S, hd, 10000.0))
    layer.fill_synthetic(1, 0.02, 0.02)
    rms = dev(np.ones(d, np.float32))
    L = mh.lib()
    try:
        B, N = 2048, 64                                     # 2^17 rows, 2^31 hidden values
        x = rng.standard_normal((B * N, d)).astype(np.float32)
        dx, par, pos = dev(x), dev(make_parents("chain", B, N, 0)), dev(np.zeros(B, np.int32))
        cache = [mh.DeviceArray((B * N, S, nkv * hd)) for _ in range(2)]
        draft = [mh.DeviceArray((B, N, nkv * hd)) for _ in range(2)]
        for t in cache + draft:
            t.zero()
        kv, kvd = [t.ptr for t in cache], [t.ptr for t in draft]
        rows = dev(np.zeros(B * N, np.int32))
        assert L.moe_hip_tree_block_dev(at.h, layer.h, rms.ptr, dx.ptr, B, N, par.ptr, pos.ptr, *kv, *kvd, EPS, None, None, None) == 2
        assert L.moe_hip_decode_block_dev(at.h, layer.h, rms.ptr, dx.ptr, B * N, rows.ptr, *kv, EPS, None, None, None) == 2
        mh.synchronize()
        assert np.array_equal(dx.to_host(), x)
        assert not any(t.to_host().any() for t in draft + cache)
        B = 1000
        at.tree_dev(dx.ptr, mh.DeviceArray((B * N, d)).ptr, B, N, par.ptr, pos.ptr, *kv, *kvd, EPS)   # (its own workspace)
        for t in draft:
            t.zero()
        big = mh.Layer(d, 16384, 2, 2)                      # (8 GB of hidden values)
        big.fill_synthetic(1, 0.02, 0.02)
        with mh.Graph() as g:
            mh.fill_normal_dev(rms.ptr, 4, 1, 0, 1.0, 0.0)
        try:
            norm = mh.DeviceArray((B * N, d))
            assert L.moe_hip_tree_block_dev(at.h, big.h, rms.ptr, dx.ptr, B, N, par.ptr, pos.ptr, *kv, *kvd, EPS,
                                            norm.ptr, None, None) == 1
            mh.synchronize()
            assert np.array_equal(dx.to_host(), x) and not any(t.to_host().any() for t in draft)
        finally:
            g.close()
            big.close()
    finally:
        at.close()
        layer.close()


def test_commit_refuses_launches_past_the_grid_without_gpu():
    """Drafts of more float4s than a launch has threads are refused, before
    anything touches a device."""
    L, P = mh.lib(), C.c_void_p
    arrs = [(P * 1)(v << 44) for v in range(1, 5)]
    for B, N, kd in ((8192, 64, 32768), (1 << 19, 1, 32768), (1, 64, 2147483644)):
        assert L.moe_hip_tree_commit_dev(1, *arrs, B, N, kd, 8, P(4096), P(1 << 30), P(1 << 31), None, None) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("block", range(10))
def test_random_drafted_shapes(block):
    """Seeded random shapes of attention (head shapes, widths, trees, positions
    inside and outside the cache, small and large calls) and of verification
    (vocabularies up to 90000), ten of each."""
    for seed in range(5000 + 10 * block, 5010 + 10 * block):
        rng = np.random.default_rng(seed)
        nkv, G, hd = int(rng.integers(1, 5)), int(rng.integers(1, 9)), 8 * int(rng.integers(1, 9))
        N = int(rng.integers(1, 65)) if rng.random() < 0.6 else int(rng.integers(1, 9))
        B = int(np.exp(rng.uniform(0, np.log(max(2, min(200, 1500 // N))))))
        d = 4 * int(rng.integers(2, 100))
        S = int(np.exp(rng.uniform(np.log(2), np.log(700 if B * N < 400 else 150))))
        kind = rng.choice(["chain", "tree", "forest", "holes", "ragged", "star", "none"])
        pos = rng.integers(-1 if rng.random() < 0.3 else 0, S + (1 if rng.random() < 0.3 else 0), B)
        many = "many" if rng.random() < 0.6 and N * nkv * hd * 4 * (2 ** 22 // max(1, B * N * nkv * G)) * B < 3e8 else "few"
        print(f"[gpu-test] seed {seed}: tree {(B, N, d, nkv * G, nkv, hd, S)} {kind} {many}", flush=True)
        check_tree(*tree_case(B, N, d, nkv * G, nkv, hd, S, pos, seed, kind, many), nkv * G, nkv, hd, in_place=bool(rng.random() < 0.3))
        V = int(np.exp(rng.uniform(0, np.log(90000))))
        B = int(rng.integers(1, max(2, min(80, 3000000 // (V * min(N, 20))))))
        N = min(N, 20) if V > 2000 else N
        probs, kind = bool(rng.random() < 0.7), rng.choice(["chain", "tree", "forest", "holes", "ragged", "star"])
        print(f"[gpu-test] seed {seed}: verify {(B, N, V)} {kind} {probs}", flush=True)
        check_verify(*verify_case(B, N, V, kind, seed, probs, float(rng.uniform(0.2, 4))), pad=int(rng.integers(0, 4)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(12, 10, 300), (3, 14, 9000), (4, 8, 70001), (64, 4, 66000)], ids=lambda s: "_".join(map(str, s)))
def test_tree_verify_no_numbers_in_q(shape):
    """Entries of q that are negative or NaN count as 0, like p's: nothing is
    taken off a token there, in the first pass over a row and in those from
    lists."""
    B, N, V = shape
    print(f"[gpu-test] verify no numbers in q {shape}", flush=True)
    p, q, par, tok, ua, us = verify_case(B, N, V, "star", 23)
    ua = np.maximum(ua, 0.9).astype(np.float32)
    q[:, :, 3::40] = -0.25
    q[:, :, 5::40] = np.nan
    q[:, :, 7::90] = -np.inf
    p[:, :, 11::80] = -0.5                       # (both negative)
    q[:, :, 11::80] = -0.4
    p[:, :, 13::80] = np.nan
    q[:, :, 13::80] = -0.3
    for t in (tok, np.where(np.arange(N) % 3 == 2, tok // 40 * 40 + 3, tok), np.where(np.arange(N) % 3 == 1, tok // 40 * 40 + 5, tok)):
        check_verify(p, q, par, np.minimum(t, V - 1).astype(np.int32), ua, us)


def test_commit_refuses_overlaps_with_whole_numbers_without_gpu():
    """Caches over positions, paths or counts, and positions written over
    drafts or caches, are refused."""
    L, P = mh.lib(), C.c_void_p
    B, N, kd, S = 4, 8, 16, 10                      # drafts of 2 KB, caches of 2.5 KB

    def commit(kc=0x30000, vc=0x40000, kdr=0x50000, vdr=0x60000, pos=0x10000, path=0x11000, n_acc=0x12000, out=0x13000):
        arrs = [(P * 2)(a, a + 0x100000) for a in (kdr, vdr, kc, vc)]
        return L.moe_hip_tree_commit_dev(2, *arrs, B, N, kd, S, P(pos), P(path), P(n_acc), P(out), None)

    for what in ("pos", "path", "n_acc"):
        for at in (0x30000, 0x30000 + 2556, 0x40010, 0x130020, 0x140020):
            assert commit(**{what: at}) == 1, (what, hex(at))
    for at in (0x30000, 0x40010, 0x50000 + 2044, 0x60000, 0x130020, 0x150020):
        assert commit(out=at) == 1, hex(at)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 3, 4, 8, 12, 40])
def test_attn_tree_values_near_the_largest(N, positions):
    """Cached values of 1e37 and scores that grow along the context: sums before
    the division stay finite in every block size, outputs are the definition's
    (W_O = 1e-37)."""
    B, nh, nkv, hd, S = 3, 8, 2, 64, 330
    x, w, kc, vc, pos, c, s, par = tree_case(B, N, 512, nh, nkv, hd, S, [250, 130, 40], 180 + N, "tree", positions)
    w["wo"] = (1e-37 * np.eye(512)).astype(np.float32)
    ramp = np.linspace(0.02, 1.0, S, dtype=np.float32)[:, None]
    kc[:, :S] *= ramp
    vc[:, :S] *= np.float32(3e37)
    vc[1, :S] = np.float32(3.4e38) * np.sign(vc[1, :S])
    print(f"[gpu-test] values near the largest N={N}", flush=True)
    got = run_tree(x, w, kc, vc, pos, c, s, par, nh, nkv, hd)
    y, _, _, live = to.attend(x, (w["wq"], w["wk"], w["wv"], w["wo"]), w["rms"], EPS, c, s, par, pos, kc, vc, nh, nkv, hd)
    assert live.all() and np.isfinite(got[0]).all()
    for b in range(B):
        assert orc.rel_l2(got[0][b].astype(np.float64) - x[b], y[b] - x[b]) <= 1e-5, b
