"""GPU tests of generation over a paged KV cache: tree attention, verification
of drafted tokens, committing and forking sequences.

Attention is compared with a 64-bit computation of the same formula on the same
rounded inputs. Its error bound is the formula's: with A = sum_j p_j |v_j|, u
the unit roundoff of the dtype and e the error of a score, rounding the
probabilities to the dtype (16-bit types) and the result once gives at most
u (A + |o|), a score's error moves p by a factor of at most 1 + 2 e, and
probabilities below the smallest fp16 number vanish. Verification and the page
operators give whole numbers and copies: they have to be equal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


@pytest.fixture(autouse=True)
def _clean_error_word(dev):
    """Every test must leave the device error word at 0 (those that set it read and clear it)."""
    yield
    from fxb200 import _lib
    code = _lib.device_error(clear=True)
    assert code == 0, f"device error word {code}"


# ------------------------------------------------------------------ tree attention
def random_tree(B, T, rng):
    par = np.full((B, T), -1, np.int32)
    for b in range(B):
        for i in range(1, T):
            par[b, i] = rng.randint(max(0, i - 4), i)
    return torch.from_numpy(par)


def make(dev, dtype, B, T, Hq, Hkv, D, lens, page, seed, n_nodes=None, layout="fused", spread=1.5):
    from fxlm import tree_masks
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=dev, dtype=F32)

    held = [-(-(n + T) // page) for n in lens]
    W = max(held) + 1
    P = sum(held) + 2
    order = rng.permutation(P)[:sum(held)]
    table, at = np.full((B, W), -1, np.int32), 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    if layout == "nhd":  # (P, page, H, D) storage seen as (P, H, page, D); separate q, k, v
        kp, vp = (randn(P, page, Hkv, D).to(dtype).transpose(1, 2) for _ in range(2))
        q, k, v = ((randn(B, T, h, D) * spread).to(dtype) for h in (Hq, Hkv, Hkv))
    else:  # keys and values interleaved in one pool; q, k, v slices of one projection
        pool = randn(P, Hkv, 2, page, D).to(dtype)
        kp, vp = pool[:, :, 0], pool[:, :, 1]
        qkv = (randn(B, T, Hq + 2 * Hkv, D) * spread).to(dtype)
        q, k, v = qkv.split([Hq, Hkv, Hkv], dim=2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    n_nodes = [T] * B if n_nodes is None else n_nodes
    return dict(q=q, k=k, v=v, k_pages=kp, v_pages=vp, page_table=torch.from_numpy(table).to(dev),
                ctx_lens=i32(lens), n_nodes=i32(n_nodes), tree_mask=tree_masks(random_tree(B, T, rng)).to(dev))


def attention_64(a, scale=None):
    """(o, bound of the error) by the formula in 64 bits, one node at a time."""
    q, k, v, kp, vp = (a[n] for n in ("q", "k", "v", "k_pages", "v_pages"))
    B, T, Hq, D = q.shape
    Hkv, page = k.shape[2], kp.shape[2]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    u = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}[q.dtype]
    p_round = 0.0 if q.dtype == F32 else 1.0
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for b in range(B):
        n, L = int(a["n_nodes"][b]), int(a["ctx_lens"][b])
        pages = a["page_table"][b, :-(-L // page)].long()
        for t in range(n):
            m = int(a["tree_mask"][b, t])
            see = [j for j in range(n) if (m >> j) & 1]
            for h in range(Hkv):
                kk = torch.cat([kp[pages, h].reshape(-1, D)[:L], k[b, see, h]]).double()
                vv = torch.cat([vp[pages, h].reshape(-1, D)[:L], v[b, see, h]]).double()
                if not len(kk):
                    continue
                qq = q[b, t, h * G:(h + 1) * G].double()
                p = torch.softmax(qq @ kk.T * scale, -1)
                r, A = p @ vv, p @ vv.abs()
                e = D * 2.0 ** -23 * float((qq.abs() @ kk.abs().T).max()) * scale + 2.0 ** -20
                low = 2.0 ** -24 * len(kk) * vv.abs().max() if q.dtype == F16 else 0.0
                o[b, t, h * G:(h + 1) * G] = r
                tol[b, t, h * G:(h + 1) * G] = 1.02 * u * (p_round * A + r.abs()) + 2 * e * A + low
    return o, tol


def check(a, scale=None, **kw):
    from fxlm import tree_attention
    ref, tol = attention_64(a, scale)
    before = a["k_pages"].clone(), a["v_pages"].clone()
    o = tree_attention(**a, scale=scale, **kw)
    torch.cuda.synchronize()
    bad = (o.double() - ref).abs() > tol
    assert torch.isfinite(o).all()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((o.double() - ref).abs() / (tol + 1e-30)).max()}"
    # the nodes' keys and values stand behind the sequences, nothing else changed
    page = a["k_pages"].shape[2]
    for pool, was, new in ((a["k_pages"], before[0], a["k"]), (a["v_pages"], before[1], a["v"])):
        for b in range(a["q"].shape[0]):
            for j in range(int(a["n_nodes"][b])):
                at = int(a["ctx_lens"][b]) + j
                was[int(a["page_table"][b, at // page]), :, at % page] = new[b, j]
        assert torch.equal(pool.view(torch.int16 if pool.element_size() == 2 else torch.int32),
                           was.view(torch.int16 if pool.element_size() == 2 else torch.int32))
    return o


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,lens,page", [
    (1, 1, 1, 1, 64, [0], 16),                       # one token, empty cache
    (1, 1, 12, 12, 64, [1], 16),
    (2, 1, 4, 2, 128, [15, 16], 16),                 # the node opens a page, or not
    (3, 2, 3, 1, 64, [17, 127, 128], 32),
    (4, 5, 12, 12, 64, [63, 64, 65, 0], 64),
    (2, 7, 8, 1, 128, [255, 257], 128),
    (2, 16, 10, 5, 64, [1000, 31], 16),
    (3, 17, 6, 2, 128, [129, 640, 5], 256),
    (2, 33, 8, 2, 64, [511, 70], 64),
    (1, 64, 16, 2, 128, [300], 32),                  # 512 rows on a key head
    (2, 64, 2, 2, 64, [1, 900], 128),
    (9, 3, 7, 7, 128, [0, 1, 2, 3, 100, 200, 300, 33, 8], 16),
])
def test_attention_shapes(dev, dtype, B, T, Hq, Hkv, D, lens, page):
    check(make(dev, dtype, B, T, Hq, Hkv, D, lens, page, seed=B * 100 + T))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G,Hkv,D,L", [(1, 1, 2, 64, 9001), (2, 4, 1, 128, 20011), (9, 8, 2, 128, 5003),
                                         (64, 1, 3, 64, 4099)])
def test_attention_long(dev, dtype, T, G, Hkv, D, L):
    check(make(dev, dtype, 1, T, Hkv * G, Hkv, D, [L], 64, seed=T))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,Hq,Hkv", [(5, 4, 4), (24, 8, 2)])
def test_attention_uneven_rows_and_layout(dev, dtype, T, Hq, Hkv):
    # lengths from none to long, rows with fewer nodes and with none; pages stored token-major
    a = make(dev, dtype, 6, T, Hq, Hkv, 64, [0, 3000, 1, 77, 512, 129], 32, seed=3,
             n_nodes=[T, 1, 0, T - 1, 2, T], layout="nhd")
    o = check(a)
    for b, n in enumerate(a["n_nodes"].tolist()):
        assert not o[b, n:].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G", [(6, 1), (40, 4)])
def test_attention_masks(dev, dtype, T, G):
    # masks that are no trees: rows that see nothing, only a later node, everything, bit 63 of T=64 trees
    a = make(dev, dtype, 3, T, 2 * G, 2, 64, [0, 5, 200], 16, seed=5)
    g = torch.Generator().manual_seed(1)
    m = torch.randint(-(2 ** 62), 2 ** 62, (3, T), generator=g)
    m[:, 0] = 0
    m[:, 1] = 1 << (T - 1)
    m[:, 2] = -1
    a["tree_mask"] = m.to(dev)
    o = check(a)
    assert not o[0, 0].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G,D", [(4, 1, 64), (4, 8, 128), (30, 4, 128)])
def test_attention_hidden_values(dev, dtype, T, G, D):
    # infinities and NaN where no visible key is: behind the sequences, in nodes that do not
    # exist, and in a node that only its own branch sees
    B, lens = 3, [0, 70, 333]
    clean = make(dev, dtype, B, T, G * 2, 2, D, lens, 32, seed=11, n_nodes=[T - 1] * B)
    ref, tol = attention_64(clean)
    a = dict(clean, k_pages=clean["k_pages"].clone(), v_pages=clean["v_pages"].clone(),
             q=clean["q"].clone(), k=clean["k"].clone(), v=clean["v"].clone())
    page = 32
    for pool, bad in ((a["k_pages"], float("nan")), (a["v_pages"], float("inf"))):
        for b in range(B):
            held = a["page_table"][b][a["page_table"][b] >= 0].long()
            for slot in range(lens[b], len(held) * page):
                pool[held[slot // page], :, slot % page] = bad
        free = sorted(set(range(pool.shape[0])) - set(a["page_table"].flatten().tolist()))
        pool[free] = bad
    for x in (a["q"], a["k"], a["v"]):
        x[:, T - 1] = float("nan")
    hide = 1  # node 1: only itself and its descendants see it
    a["k"][:, hide] = float("inf")
    a["v"][:, hide] = float("-inf")
    a["v"][:, hide, :, 3] = float("nan")
    from fxlm import tree_attention
    o = tree_attention(**a).double()
    sees = ((a["tree_mask"] >> hide) & 1).bool()
    sees[:, T - 1] = False
    assert not sees[:, 0].any() and sees[:, hide].all()
    assert ((o - ref).abs() <= tol)[~sees].all()
    assert not torch.isfinite(o[sees]).any(-1).all()


def test_attention_value_infinity_reaches_who_sees_it(dev):
    # an infinite value in a visible node, with finite keys: the formula's infinity in that element alone
    from fxlm import tree_attention
    for dtype in (BF16, F32):
        for T, G in ((4, 1), (30, 4)):
            a = make(dev, dtype, 1, T, 2 * G, 2, 64, [50], 32, seed=2)
            a["v"] = a["v"].clone()
            ref, tol = attention_64(a)
            a["v"][0, 1, :, 5] = float("inf")
            o = tree_attention(**a).double()
            sees = ((a["tree_mask"][0] >> 1) & 1).bool()
            hit = torch.zeros_like(o, dtype=torch.bool)
            hit[0, sees, :, 5] = True
            assert (o[hit] == float("inf")).all()
            assert ((o - ref).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G", [(3, 1), (20, 8)])
def test_attention_peaked_scores(dev, dtype, T, G):
    # large scores whose maximum rises along the sequence: every rescaling of the running sums is taken
    a = make(dev, dtype, 1, T, G, 1, 64, [777], 64, seed=4)
    pages, page = a["page_table"][0].long(), 64
    up = torch.linspace(0, 24, 777, device=dev)
    for j in range(777):
        a["k_pages"][pages[j // page], :, j % page] = (a["k_pages"][pages[j // page], :, j % page].float()
                                                       * 0.1 + up[j]).to(dtype)
    a["q"] = torch.full_like(a["q"], 0.125)
    check(a)
    check(a, scale=0.5)


def test_attention_no_dependence_on_the_past(dev):
    # the same call twice is the same result bit for bit, other calls in between or not
    from fxlm import tree_attention
    a = make(dev, BF16, 5, 6, 8, 2, 128, [3000, 1, 700, 64, 9000], 64, seed=1)
    b = make(dev, BF16, 2, 64, 8, 1, 64, [2000, 900], 16, seed=2)
    first = tree_attention(**a).clone()
    for _ in range(3):
        tree_attention(**b)
        assert torch.equal(tree_attention(**a), first)


def test_attention_other_stream_and_graph(dev):
    from fxb200 import ops
    from fxlm import tree_attention
    a = make(dev, BF16, 3, 4, 8, 8, 64, [500, 900, 3], 32, seed=6)
    want = tree_attention(**a).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree_attention(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    ws = {}
    with ops.graph_workspaces(ws), torch.cuda.graph(g):
        out = tree_attention(**a)
    for _ in range(3):
        out.zero_()
        g.replay()
        tree_attention(**a)
        assert torch.equal(out, want)
    # lengths are read on the device: a replay after they changed is the new result
    a["ctx_lens"].copy_(torch.tensor([17, 880, 0], dtype=torch.int32))
    g.replay()
    assert torch.equal(out, tree_attention(**a))


@pytest.mark.parametrize("T,G,dtype", [(2, 1, BF16), (32, 1, BF16), (2, 1, F32)])
def test_attention_far_pages(dev, T, G, dtype):
    # pages beyond 2^32 bytes and 2^31 elements of the pool
    page, D, H = 64, 128, 4
    P = 2 ** 31 // (page * D * H) + 40
    pool = torch.zeros(P, H, page, D, device=dev, dtype=dtype)
    a = make(dev, dtype, 2, T, H * G, H, D, [150, 1], page, seed=8)
    far = torch.arange(P - 10, P, device=dev)
    near = a["page_table"].clone()
    for k in ("k_pages", "v_pages"):
        src = a[k]
        one = pool if k == "k_pages" else pool.clone()
        for i in range(src.shape[0]):
            one[far[i]] = src[i]
        a[k] = one
    a["page_table"] = torch.where(near >= 0, (near + P - 10).int(), -1).int()
    ref, tol = attention_64(a)
    from fxlm import tree_attention
    o = tree_attention(**a)
    assert ((o.double() - ref).abs() <= tol).all()
    assert torch.equal(a["k_pages"][int(a["page_table"][1, 0]), :, 1], a["k"][1, 0])


def test_attention_pages_that_do_not_fit(dev):
    from fxb200 import _lib
    from fxlm import tree_attention
    a = make(dev, BF16, 2, 3, 4, 4, 64, [40, 20], 16, seed=9)
    good = tree_attention(**a)
    for change in ({"page_table": torch.where(a["page_table"] == a["page_table"][0, 1], 10 ** 6, a["page_table"]).int()},
                   {"page_table": torch.where(a["page_table"] == a["page_table"][0, 1], -5, a["page_table"]).int()},
                   {"ctx_lens": torch.tensor([10 ** 8, 20], dtype=torch.int32, device=dev)},
                   {"ctx_lens": torch.tensor([-3, 20], dtype=torch.int32, device=dev)},
                   {"n_nodes": torch.tensor([70, 3], dtype=torch.int32, device=dev)}):
        o = tree_attention(**dict(a, **change))
        assert torch.equal(o[1], good[1])
        with pytest.raises(RuntimeError, match="KV cache"):
            _lib.raise_on_device_error()


# ------------------------------------------------------------------ verification
def verify_plain(tokens, par, n, p, u, q):
    """One row, one step at a time: fp32 for single values, Python integers for sums."""
    f = np.float32

    def fixed(w):
        return int(min(w, f(1)) * f(2 ** 36)) if w > 0 else 0

    def fixed_row(w):
        w = np.where(w > 0, w, f(0)).clip(max=f(1))
        return (w * f(2 ** 36)).astype(np.int64)

    V = p.shape[1]
    if n == 0:
        return [], -1
    path, cur = [0], 0
    w, scale, mass, empty = p[0].copy(), f(1), f(1), False
    for c in range(1, n):
        if par[c] != cur or empty:
            continue
        x = int(tokens[c])
        inside = 0 <= x < V
        a = w[x] if inside and w[x] > 0 else f(0)
        if q is None:
            a = min(a, f(1))
            take = f(u[c]) * mass < a
        else:
            take = f(u[c]) * (q[cur][x] if inside else f(0)) < a * scale
        if take:
            cur = c
            path.append(c)
            w, scale, mass = p[c].copy(), f(1), f(1)
        elif q is None:
            mass = max(mass - a, f(0))
            if inside:
                w[x] = 0
        else:
            w = w * scale - q[cur]
            w = np.where(w > 0, w, f(0))
            total = int(fixed_row(w).sum())
            if total:
                scale = f(1) / (f(total) * f(2.0 ** -36))
            else:
                empty = True
    fr = fixed_row(w)
    if fr.sum() == 0:
        fr = fixed_row(p[cur])
    total = int(fr.sum())
    if total == 0:
        return path, -1
    thr = (total * int(min(max(u[0], 0), 1 - 2.0 ** -24) * 2 ** 24)) >> 24
    return path, int(np.searchsorted(np.cumsum(fr), thr, side="right"))


def verify_inputs(B, T, V, draft, seed, chain=False, peak=3.0):
    rng = np.random.RandomState(seed)
    par = random_tree(B, T, rng).numpy()
    if chain:
        par[:, 1:] = np.arange(T - 1)
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, T, V, generator=g) * peak
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits * 0.7 + torch.randn(B, T, V, generator=g), -1)
    src = (q if draft else p).double().numpy()
    tokens = np.zeros((B, T), np.int64)
    for b in range(B):
        for c in range(1, T):
            w = src[b, par[b, c]]
            tokens[b, c] = rng.choice(V, p=w / w.sum())
    u = torch.rand(B, T, generator=g)
    n = rng.randint(0, T + 1, B).astype(np.int32)
    n[0] = T
    return torch.from_numpy(tokens), torch.from_numpy(par), torch.from_numpy(n), p, u, (q if draft else None)


def verify_check(dev, tokens, par, n, p, u, q):
    from fxlm import verify_tree
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    path, n_path, nxt = verify_tree(to(tokens), to(par), to(n), to(p), to(u), draft_probs=to(q))
    lengths = []
    for b in range(tokens.shape[0]):
        want, tok = verify_plain(tokens[b].numpy(), par[b].numpy(), int(n[b]), p[b].numpy(), u[b].numpy(),
                                 None if q is None else q[b].numpy())
        got = path[b].tolist()
        assert got == want + [-1] * (tokens.shape[1] - len(want)), (b, got, want)
        assert int(n_path[b]) == len(want) and int(nxt[b]) == tok, (b, int(nxt[b]), tok)
        lengths.append(len(want))
    return lengths


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("B,T,V,chain", [(1, 1, 5, False), (1, 2, 33, True), (7, 9, 257, True), (16, 33, 1000, False),
                                         (5, 64, 4097, False), (3, 8, 32768, True), (2, 5, 50257, False),
                                         (2, 3, 131075, False), (70, 4, 100, False)])
def test_verify(dev, B, T, V, chain, draft):
    lengths = verify_check(dev, *verify_inputs(B, T, V, draft, seed=B * T + V, chain=chain))
    if B * T > 60 and T > 2:
        assert max(lengths) > 1 and min(lengths) <= 1


def test_verify_many_rejections(dev):
    # drafts that the target hardly ever takes: long chains of residuals, and rows whose children all fail
    tokens, par, n, p, u, q = verify_inputs(12, 20, 300, True, seed=4)
    par[:, 1:] = 0
    g = torch.Generator().manual_seed(9)
    q = torch.softmax(torch.randn(12, 20, 300, generator=g) * 2, -1)
    tokens = torch.multinomial(q[:, 0], 20, replacement=True, generator=g)
    verify_check(dev, tokens, par, torch.full_like(n, 20), p, u, q)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_degenerate_rows(dev, draft):
    B, T, V = 8, 4, 70
    tokens, par, n, p, u, q = verify_inputs(B, T, V, draft, seed=6)
    n[:] = T
    par[:, 1:] = 0
    p[0] = 0                                     # no mass at all
    p[1] = float("nan")
    p[2] = 0; p[2, :, 69] = 1                    # everything on the last token
    p[3] = 0; p[3, :, 0] = 1
    tokens[4, 1:] = torch.tensor([-1, V, 2 ** 40])   # tokens outside the vocabulary
    tokens[5, 1:] = tokens[5, 1]                 # the same draft three times
    p[5] = p[5, :, torch.randperm(V)]
    u[6] = 0
    u[7] = 1 - 2.0 ** -24
    if draft:
        q[5] = p[5]                              # residuals that are empty up to rounding
        q[2] = 0; q[2, :, 69] = 1
    verify_check(dev, tokens, par, n, p, u, q)
    # parents that point forward or outside are never reached
    par[0, 1:] = torch.tensor([5, -7, 3])
    verify_check(dev, tokens, par, n, p, u, q)


def test_verify_strided_rows(dev):
    from fxlm import verify_tree
    tokens, par, n, p, u, q = verify_inputs(4, 6, 333, True, seed=3)
    both = torch.empty(4, 6, 2, 340)
    both[:, :, 0, 3:336], both[:, :, 1, 3:336] = p, q
    both = both.to(dev)
    want = verify_tree(tokens.to(dev), par.to(dev), n.to(dev), p.to(dev), u.to(dev), draft_probs=q.to(dev))
    got = verify_tree(tokens.to(dev), par.to(dev), n.to(dev), both[:, :, 0, 3:336], u.to(dev),
                      draft_probs=both[:, :, 1, 3:336])
    for x, y in zip(want, got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_keeps_the_target_distribution(dev, draft):
    # the token after the root (accepted draft or drawn) follows the target, whatever was drafted:
    # 5 standard deviations of a binomial count, over 8 tokens
    from fxlm import verify_tree
    B, T, V = 40000, 4, 8
    g = torch.Generator(device=dev).manual_seed(5)
    p0 = torch.softmax(torch.randn(V, generator=g, device=dev) * 1.5, -1)
    q0 = torch.softmax(torch.randn(V, generator=g, device=dev) * 1.5, -1)
    par = torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device=dev).expand(B, T).contiguous()
    tokens = torch.multinomial(q0.expand(B, V), T, replacement=True, generator=g)
    if not draft:
        tokens[:, 1:] = torch.topk(q0, 3).indices
    p = p0.expand(B, T, V)
    path, n_path, nxt = verify_tree(tokens, par, torch.full((B,), T, dtype=torch.int32, device=dev),
                                    p, torch.rand(B, T, generator=g, device=dev),
                                    draft_probs=q0.expand(B, T, V) if draft else None)
    first = torch.where(n_path > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    count = torch.bincount(first, minlength=V).double()
    sigma = (B * p0.double() * (1 - p0.double())).sqrt()
    assert ((count - B * p0.double()).abs() <= 5 * sigma).all()
    assert (n_path > 1).float().mean() > 0.2


# ------------------------------------------------------------------ pages
class PlainPages:
    """The page table as lists, one row and one page at a time."""

    def __init__(self, c):
        self.k, self.v = c["k"].clone(), c["v"].clone()
        self.W, self.page = c["table"].shape[1], c["page"]
        self.lens = c["lens"].tolist()
        self.rows = [c["table"][s, :h].tolist() for s, h in enumerate(c["n_pages"].tolist())]
        self.ref = c["ref"].tolist()

    def free(self):
        return [p for p, r in enumerate(self.ref) if r == 0]

    def commit(self, path, n_path, room):
        P = self.page
        for s, row in enumerate(self.rows):
            n = n_path[s] if path is not None else 0
            for i in range(n):
                a, b = self.lens[s] + path[s][i], self.lens[s] + i
                for x in (self.k, self.v):
                    x[:, row[b // P], :, b % P] = x[:, row[a // P], :, a % P].clone()
            self.lens[s] += n
        want = [max(0, min(self.W, -(-(self.lens[s] + r) // P)) - len(self.rows[s])) if r > 0 else 0
                for s, r in enumerate(room)]
        free = self.free()
        if sum(want) > len(free):
            return False
        for s, w in enumerate(want):
            for _ in range(w):
                p = free.pop(0)
                self.rows[s].append(p)
                self.ref[p] = 1
        return True

    def fork(self, parents):
        P, free = self.page, self.free()
        kept = {p for s, p in enumerate(parents) if p == s}
        rows, lens = [], []
        copies = []
        for s, p in enumerate(parents):
            n = self.lens[p] if p >= 0 else 0
            row = list(self.rows[p][:-(-n // P)]) if p >= 0 else []
            if n % P and p != s:
                if p in kept:
                    if not free:
                        return False
                    new = free.pop(0)
                    copies.append((row[-1], new, n % P))
                    row[-1] = new
                else:
                    kept.add(p)
            rows.append(row)
            lens.append(n)
        for a, b, n in copies:
            for x in (self.k, self.v):
                x[:, b, :, :n] = x[:, a, :, :n]
        self.rows, self.lens = rows, lens
        self.ref = [0] * len(self.ref)
        for row in rows:
            for p in row:
                self.ref[p] += 1
        return True


def cache(dev, dtype, S, L, H, D, page, lens, extra, P=None, seed=0, W=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed)
    held = [-(-(n + extra) // page) for n in lens]
    P = sum(held) + S + 4 if P is None else P
    W = max(held) + 5 if W is None else W
    order, at = rng.permutation(P), 0
    table, ref = np.full((S, W), -1, np.int32), np.zeros(P, np.int32)
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        ref[order[at:at + h]] = 1
        at += h
    both = torch.randn(L, P, 2, H, page, D, generator=g, device=dev).to(dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(k=both[:, :, 0], v=both[:, :, 1], table=torch.from_numpy(table).to(dev), n_pages=i32(held),
                lens=i32(lens), ref=torch.from_numpy(ref).to(dev), page=page)


def same(c, want, lens):
    torch.cuda.synchronize()
    assert lens.tolist() == want.lens
    assert c["n_pages"].tolist() == [len(r) for r in want.rows]
    assert c["ref"].tolist() == want.ref
    W = want.W
    assert c["table"].tolist() == [r + [-1] * (W - len(r)) for r in want.rows]
    assert torch.equal(c["k"], want.k) and torch.equal(c["v"], want.v)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("S,L,H,D,page,lens,T", [
    (1, 1, 1, 64, 16, [0], 1), (1, 3, 2, 64, 16, [15], 8), (4, 2, 3, 128, 32, [0, 31, 32, 100], 9),
    (3, 12, 12, 64, 16, [500, 7, 64], 64), (6, 1, 5, 8, 64, [1, 2, 3, 63, 64, 65], 17),
    (2, 2, 2, 128, 256, [250, 300], 33)])
def test_commit(dev, dtype, S, L, H, D, page, lens, T):
    from fxlm import kv_commit
    rng = np.random.RandomState(T)
    c = cache(dev, dtype, S, L, H, D, page, lens, T, seed=T)
    want = PlainPages(c)
    n = [int(rng.randint(0, T + 1)) for _ in range(S)]
    n[-1] = T if S > 1 else n[-1]
    path = [sorted(rng.permutation(T)[:k].tolist()) + [-1] * (T - k) for k in n]
    room = [int(rng.choice([0, 1, page, 3 * page])) for _ in range(S)]
    room[0] = T
    assert want.commit(path, n, room)
    old = c["lens"].clone()
    lens_out = kv_commit(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"],
                         torch.tensor(path, dtype=torch.int32, device=dev),
                         torch.tensor(n, dtype=torch.int32, device=dev),
                         room=torch.tensor(room, dtype=torch.int32, device=dev))
    same(c, want, lens_out)
    assert torch.equal(c["lens"], old)


@pytest.mark.parametrize("S,P", [(1, 5), (600, 4000), (3, 70001)])
def test_reserve(dev, S, P):
    from fxlm import kv_reserve
    rng = np.random.RandomState(S)
    lens = [int(rng.randint(0, 40)) for _ in range(S)] if S > 1 else [0]
    c = cache(dev, BF16, S, 1, 1, 8, 16, lens, 0, P=P, seed=S, W=max(5, P // 10))
    want = PlainPages(c)
    room = [int(rng.randint(0, 50)) for _ in range(S)] if S > 1 else [80]
    assert want.commit(None, None, room)
    kv_reserve(c["table"], c["n_pages"], c["lens"], c["ref"], torch.tensor(room, dtype=torch.int32, device=dev), 16)
    same(c, want, c["lens"])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("S,L,H,D,page,lens,parents", [
    (1, 1, 1, 64, 16, [5], [0]), (2, 2, 3, 64, 16, [5, 40], [1, 1]), (2, 1, 1, 64, 16, [0, 16], [1, 0]),
    (5, 3, 2, 128, 32, [33, 64, 7, 0, 100], [4, 4, 0, 2, 2]), (4, 2, 2, 64, 128, [100, 300, 128, 5], [1, 2, 3, 0]),
    (6, 12, 12, 64, 16, [500, 3, 9, 77, 16, 1], [0, 0, -1, 0, 3, -1]), (3, 1, 1, 8, 256, [1, 2, 3], [-1, -1, -1])])
def test_fork(dev, dtype, S, L, H, D, page, lens, parents):
    from fxlm import kv_fork
    c = cache(dev, dtype, S, L, H, D, page, lens, 3, seed=S + L)
    want = PlainPages(c)
    par = torch.tensor(parents, dtype=torch.int32, device=dev)
    for _ in range(3):  # forks of forks: shared pages, freed pages that come back
        assert want.fork(parents)
        kv_fork(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"], par)
        same(c, want, c["lens"])


def test_fork_many_rows(dev):
    from fxlm import kv_fork
    rng = np.random.RandomState(2)
    S = 700
    c = cache(dev, BF16, S, 2, 1, 16, 16, [int(rng.randint(0, 60)) for _ in range(S)], 2, P=6000, seed=1)
    want = PlainPages(c)
    parents = [int(rng.randint(-1, S)) for _ in range(S)]
    assert want.fork(parents)
    kv_fork(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"],
            torch.tensor(parents, dtype=torch.int32, device=dev))
    same(c, want, c["lens"])


def test_calls_that_do_not_fit_change_nothing(dev):
    from fxb200 import _lib
    from fxlm import kv_commit, kv_fork, kv_reserve
    c = cache(dev, BF16, 3, 2, 2, 64, 16, [20, 30, 7], 2, P=6, seed=1, W=6)  # 5 pages held, one free
    want = PlainPages(c)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = (c["table"], c["n_pages"], c["lens"], c["ref"])

    def refused():
        with pytest.raises(RuntimeError, match="KV cache"):
            _lib.raise_on_device_error()
        same(c, want, c["lens"])

    kv_reserve(*args, i32([0, 20, 20]), 16)              # two pages wanted
    refused()
    kv_fork(c["k"], c["v"], *args, i32([0, 0, 0]))       # two copies wanted
    refused()
    kv_fork(c["k"], c["v"], *args, i32([0, 3, 2]))       # no such row
    refused()
    kv_fork(c["k"], c["v"], *args, i32([0, -2, 2]))
    refused()
    kv_reserve(*args, i32([100, 0, 0]), 16)              # longer than a row of the table: 6 - 2 pages wanted
    refused()
    for path in ([[1, 0], [0, 1], [0, 1]], [[0, 0], [0, 1], [0, 1]], [[0, 2], [0, 1], [0, 1]], [[-1, 1], [0, 1], [0, 1]]):
        kv_commit(c["k"], c["v"], *args, i32(path), i32([2, 0, 0]))
        got = c["k"].clone()
        with pytest.raises(RuntimeError, match="KV cache"):
            _lib.raise_on_device_error()
        del got
    kv_reserve(*args, i32([0, 3, 0]), 16)                # one page: fits
    assert want.commit(None, None, [0, 3, 0])
    assert c["ref"].tolist() == want.ref


def test_page_calls_in_a_graph(dev):
    from fxlm import kv_commit, kv_fork
    c = cache(dev, BF16, 3, 2, 2, 64, 16, [20, 30, 7], 8, P=40, seed=1)
    want = PlainPages(c)
    path = torch.tensor([[0, 2, 5, -1]] * 3, dtype=torch.int32, device=dev)
    n = torch.tensor([3, 2, 0], dtype=torch.int32, device=dev)
    room = torch.full((3,), 8, dtype=torch.int32, device=dev)
    par = torch.tensor([1, 1, 0], dtype=torch.int32, device=dev)
    args = (c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"])
    path8 = torch.cat([path, torch.full((3, 4), -1, dtype=torch.int32, device=dev)], 1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        new = kv_commit(*args, path8, n, room=room)
        c["lens"].copy_(new)
        kv_fork(*args, par)
    for _ in range(3):
        assert want.commit(path8.tolist(), n.tolist(), room.tolist())
        assert want.fork(par.tolist())
        # fork drops the room that commit made: give it back before the next replay
        g.replay()
        same(c, want, c["lens"])
        from fxlm import kv_reserve
        kv_reserve(c["table"], c["n_pages"], c["lens"], c["ref"], room, 16)
        want.commit(None, None, room.tolist())


@pytest.mark.parametrize("T,Hq,Hkv", [(2, 4, 2), (20, 2, 2)])
def test_attention_many_batch_rows(dev, T, Hq, Hkv):
    # more batch rows than a thread block has threads, most of them short, a third without nodes,
    # runs of idle rows at both ends; then no row with a node at all
    rng = np.random.RandomState(T)
    B = 450
    n = [0 if b < 9 or b > B - 12 or rng.rand() < 0.3 else int(rng.randint(1, T + 1)) for b in range(B)]
    lens = [int(rng.choice([0, 1, 20, 130, 300])) for _ in range(B)]
    a = make(dev, BF16, B, T, Hq, Hkv, 64, lens, 32, seed=T, n_nodes=n)
    o = check(a)
    for b in range(B):
        assert not o[b, n[b]:].any()
    from fxlm import tree_attention
    a["n_nodes"].zero_()
    assert not tree_attention(**a).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G,D", [(3, 1, 128), (7, 1, 64), (5, 3, 64), (30, 4, 128)])
def test_attention_context_infinity_leaves_empty_rows_zero(dev, dtype, T, G, D):
    # an infinite value in the context: infinity for every node, zeros still for rows that are no node's
    from fxlm import tree_attention
    a = make(dev, dtype, 2, T, 2 * G, 2, D, [200, 70], 16, seed=5, n_nodes=[1, T], spread=0.2)
    ref, tol = attention_64(a)
    for b, at in ((0, 3), (0, 150), (1, 64)):
        a["v_pages"][int(a["page_table"][b, at // 16]), :, at % 16, 9] = float("inf")
    o = tree_attention(**a).double()
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, :1, :, 9] = hit[1, :, :, 9] = True
    assert (o[hit] == float("inf")).all()
    assert ((o - ref).abs() <= tol)[~hit].all()
    assert (o[0, 1:] == 0).all()


def test_attention_plain_captures(dev):
    # graphs captured without ops.graph_workspaces: replayed in another order than captured, with larger calls
    # (whose workspaces are larger) and other allocations in between, and on two streams at once
    from fxlm import tree_attention
    few = [make(dev, BF16, 3, 4, 8, 8, 64, [500, 900, 3], 32, seed=6), make(dev, F16, 2, 2, 6, 2, 128, [4000, 70], 16, seed=7)]
    wide = make(dev, BF16, 2, 64, 8, 1, 64, [2000, 900], 16, seed=2)
    calls = few + [wide]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = []
    with torch.cuda.stream(side):  # warm-up on the stream of the captures: the small calls' eager workspace
        for a in few:
            want.append(tree_attention(**a).clone())
    side.synchronize()
    graphs, outs = [], []
    for a in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(tree_attention(**a))
    want.append(tree_attention(**wide).clone())
    for i in (2, 1, 0, 1, 2):
        outs[i].fill_(7)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            tree_attention(**wide)
            noise = [torch.full((1 << 20,), 3, dtype=torch.int32, device=dev) for _ in range(8)]
        torch.cuda.current_stream().wait_stream(side)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])
        assert all((x == 3).all() for x in noise)
    for _ in range(5):
        for out in outs[:2]:
            out.fill_(7)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_commit_lengths_when_the_pool_is_too_small(dev):
    # more rows than a thread block has threads, the first of which want more than the pool has: every length is
    # returned and every token moved, no page is handed out
    from fxb200 import _lib
    from fxlm import kv_commit
    rng = np.random.RandomState(3)
    S, T, page = 1300, 5, 16
    lens = [int(rng.randint(0, 40)) for _ in range(S)]
    held = sum(-(-(n + T) // page) for n in lens)
    c = cache(dev, BF16, S, 2, 1, 8, page, lens, T, P=held + 3, W=20, seed=3)
    want = PlainPages(c)
    n = [int(rng.randint(0, T + 1)) for _ in range(S)]
    path = [sorted(rng.permutation(T)[:k].tolist()) + [-1] * (T - k) for k in n]
    room = [250] * S
    assert not want.commit(path, n, room)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = i32([-7] * S)
    assert kv_commit(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"], i32(path), i32(n),
                     room=i32(room), out=out) is not None
    same(c, want, out)
    with pytest.raises(RuntimeError, match="KV cache"):
        _lib.raise_on_device_error()


@pytest.mark.parametrize("n", [[3, 1], [1, -1]])
def test_commit_reports_counts_outside_the_tree(dev, n):
    from fxb200 import _lib
    from fxlm import kv_commit
    c = cache(dev, BF16, 2, 1, 1, 8, 16, [4, 5], 2, seed=1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = kv_commit(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"], i32([[0, 1], [0, 1]]), i32(n))
    assert got.tolist() == [4 + min(n[0], 2), 5 + max(n[1], 0)]
    with pytest.raises(RuntimeError, match="KV cache"):
        _lib.raise_on_device_error()


def test_commit_moves_what_fits_of_a_path(dev):
    # entries of a path that do not ascend, or lie outside the tree or the row's pages, are left out, each by
    # itself; the lengths are those of the whole path; a path longer than the tree counts as the tree's length
    from fxb200 import _lib
    from fxlm import kv_commit
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    T, page, lens = 4, 16, [20, 30, 7]
    for path, n in (([[2, 1, 3, -1], [1, 2, 3, -1], [0, 0, 3, -1]], [3, 3, 3]),
                    ([[0, 2, 4, 5], [-1, 1, 3, -1], [3, 2, 1, 0]], [4, 3, 4]),
                    ([[1, 2, 3, 3], [0, 2, 3, -1], [2, -1, -1, -1]], [9, 3, -2])):
        c = cache(dev, BF16, 3, 2, 2, 64, page, lens, T, seed=1)
        want = PlainPages(c)
        for s, row in enumerate(path):
            count = min(max(n[s], 0), T)
            for i in range(count):
                p = row[i]
                if not (max(i, row[i - 1] + 1 if i else 0) <= p < T):
                    continue
                a, b = lens[s] + p, lens[s] + i
                for x in (want.k, want.v):
                    x[:, want.rows[s][b // page], :, b % page] = x[:, want.rows[s][a // page], :, a % page].clone()
            want.lens[s] += count
        got = kv_commit(c["k"], c["v"], c["table"], c["n_pages"], c["lens"], c["ref"], i32(path), i32(n))
        same(c, want, got)
        with pytest.raises(RuntimeError, match="KV cache"):
            _lib.raise_on_device_error()


def test_attention_refuses_inputs_that_need_a_gradient(dev):
    from fxlm import tree_attention
    a = make(dev, BF16, 1, 3, 4, 4, 64, [40], 16, seed=9)
    want = tree_attention(**a).clone()
    for name in ("q", "k", "v", "k_pages", "v_pages"):
        b = dict(a, **{name: a[name].detach().clone().requires_grad_()})
        with pytest.raises(ValueError, match="gradient"):
            tree_attention(**b)
        with torch.no_grad():
            assert torch.equal(tree_attention(**b), want)


@pytest.mark.parametrize("T,dtype", [(2, BF16), (2, F32), (24, BF16)])
def test_attention_one_tree_for_all_rows(dev, T, dtype):
    from fxlm import tree_attention
    a = make(dev, dtype, 5, T, 4, 2, 64, [30, 0, 7, 200, 64], 16, seed=4)
    one = a["tree_mask"][1:2]
    want = check(dict(a, tree_mask=one.repeat(5, 1))).clone()
    assert torch.equal(tree_attention(**dict(a, tree_mask=one.expand(5, T))), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_strides_of_single_entries(dev, dtype):
    # one batch row, one node, one key head: the strides of those axes are not used and may be anything
    from fxlm import tree_attention
    for T, Hq, P in ((1, 4, 3), (1, 24, 3)):
        a = make(dev, dtype, 1, T, Hq, 1, 64, [30], 32, seed=4, layout="nhd")
        want = tree_attention(**a).clone()

        def odd(t, *strides):
            return t.as_strided(t.shape, strides)

        b = dict(a, q=odd(a["q"], 7, 3, 64, 1), k=odd(a["k"], 5, 3, 1, 1), v=odd(a["v"], 3, 5, 7, 1))
        for name in ("k_pages", "v_pages"):
            b[name] = odd(a[name], a[name].stride(0), 3, 64, 1)
        assert torch.equal(tree_attention(**b), want)


def test_commit_strides_of_single_entries(dev):
    from fxlm import kv_commit, kv_fork
    c = cache(dev, BF16, 2, 1, 1, 64, 16, [5, 9], 4, seed=1)
    want = PlainPages(c)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = (c["table"], c["n_pages"], c["lens"], c["ref"])
    k, v = (x.as_strided(x.shape, (7, x.stride(1), 3, 64, 1)) for x in (c["k"], c["v"]))
    assert want.commit([[1, 3], [0, 2]], [2, 2], [0, 0])
    c["lens"].copy_(kv_commit(k, v, *args, i32([[1, 3, -1, -1], [0, 2, -1, -1]]), i32([2, 2])))
    same(c, want, c["lens"])
    assert want.fork([1, 1])
    kv_fork(k, v, *args, i32([1, 1]))
    same(c, want, c["lens"])


def test_refusals_are_value_errors(dev):
    from fxlm import kv_commit, kv_fork, kv_reserve, tree_attention, verify_tree
    a = make(dev, BF16, 2, 3, 4, 4, 64, [40, 20], 16, seed=9)

    def refused(match, **kw):
        with pytest.raises(ValueError, match=match):
            tree_attention(**dict(a, **kw))

    pages = torch.zeros(4, 4, 24, 64, dtype=BF16, device=dev)
    refused("page 24", k_pages=pages, v_pages=pages)
    refused("scale", scale=-1.0)
    refused("scale", scale=float("nan"))
    refused("aligned", q=torch.zeros(2 * 3 * 4 * 64 + 1, dtype=BF16, device=dev)[1:].view(2, 3, 4, 64))
    refused("strides", q=torch.zeros(2, 3, 4, 68, dtype=BF16, device=dev)[..., :64])
    refused("row stride", tree_mask=torch.zeros(8, dtype=torch.int64, device=dev).as_strided((2, 3), (2, 1)))
    refused("row stride", page_table=a["page_table"][:1].expand(2, -1))
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    args = (i[:, None], i, i.clone(), torch.zeros(4, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="page 24"):
        kv_reserve(*args, i, 24)
    k = torch.zeros(2, 4, 2, 16, 4, dtype=BF16, device=dev)
    with pytest.raises(ValueError, match="D=4"):
        kv_commit(k, k, *args, i[:, None], i)
    with pytest.raises(ValueError, match="D=4"):
        kv_fork(k, k, *args, i)
    p = torch.zeros(1, 1, 8, device=dev)
    with pytest.raises(ValueError, match="V=0"):
        verify_tree(i[:, None].long(), i[:, None], i, p[..., :0], p[:, :, 0])


@pytest.mark.parametrize("dtype,T,Hq,Hkv,lens", [
    (BF16, 1, 2, 1, [40, 900, 3, 300]), (BF16, 3, 2, 2, [700, 0, 130]), (F32, 2, 3, 1, [500, 64, 5]),
    (BF16, 20, 2, 1, [700, 5, 130, 0]), (F16, 33, 4, 1, [300, 129])])
@pytest.mark.parametrize("B", [33, 48, 128, 385])
def test_attention_batches(dev, dtype, T, Hq, Hkv, lens, B):
    # as many batch rows as a warp has lanes and more, up to more than a block has threads; the last row long, so
    # that few short rows are cut into whole parts
    lens = [lens[b % len(lens)] for b in range(B - 1)] + [3000]
    check(make(dev, dtype, B, T, Hq, Hkv, 64, lens, 32, seed=B + T))


@pytest.mark.parametrize("draft", [False, True])
def test_verify_reports_numbers_of_nodes_outside_the_tree(dev, draft):
    from fxb200 import _lib
    from fxlm import verify_tree
    tokens, par, n, p, u, q = (None if x is None else x.to(dev) for x in verify_inputs(3, 4, 60, draft, seed=2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    want = verify_tree(tokens, par, i32([4, 0, 2]), p, u, draft_probs=q)
    _lib.raise_on_device_error()
    got = verify_tree(tokens, par, i32([9, -3, 2]), p, u, draft_probs=q)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="KV cache"):
        _lib.raise_on_device_error()
