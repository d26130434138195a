"""CPU: refusals of the generation operators (C ABI and Python wrappers) and
the host-side helpers of fxlm.paged. No kernel runs here."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from fxb200 import _lib
    return _lib.load()


def err():
    from fxb200 import _lib
    return _lib.last_error()


def tree_args(**kw):
    from fxb200 import _lib
    a = _lib.TreeAttnArgs()
    a.dtype, a.B, a.T, a.Hq, a.Hkv, a.D, a.page, a.P, a.W, a.scale = 2, 1, 4, 4, 2, 64, 16, 8, 4, 0.125
    a.q = a.k = a.v = a.o = a.k_pages = a.v_pages = 256
    a.table = a.lens = a.n_nodes = a.mask = 256
    a.table_sb, a.mask_sb = 4, 4
    for n in ("q", "k", "v", "o"):
        for s in ("sb", "st", "sh"):
            setattr(a, f"{n}_{s}", 64)
    for n in ("kp", "vp"):
        for s in ("sp", "sh", "st"):
            setattr(a, f"{n}_{s}", 64)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def test_struct_layouts_match(lib):
    from fxb200 import _lib
    assert lib.fxb_abi_struct_size(2) == ctypes.sizeof(_lib.TreeAttnArgs)
    assert lib.fxb_abi_struct_size(3) == ctypes.sizeof(_lib.KvArgs)


@pytest.mark.parametrize("change,word", [
    (dict(D=96), "head_dim 96"), (dict(T=65), "T=65"), (dict(T=0), "T=0"), (dict(Hq=5), "Hq=5"), (dict(B=0), "B=0"),
    (dict(page=24), "page 24"), (dict(page=512), "page 512"), (dict(page=8), "page 8"), (dict(P=0), "P=0"),
    (dict(W=0), "W=0"), (dict(table_sb=3), "row stride"), (dict(mask_sb=3), "row stride"), (dict(q=264), "aligned"),
    (dict(k_pages=0), "aligned"), (dict(mask=0), "NULL"), (dict(q_sh=12), "strides"), (dict(vp_st=-64), "strides"),
    (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale")])
def test_tree_attn_refuses(lib, change, word):
    assert lib.fxb_tree_attn(ctypes.byref(tree_args(**change)), None) == -1
    assert word in err()


def test_tree_attn_refuses_dtype_and_null(lib):
    assert lib.fxb_tree_attn(ctypes.byref(tree_args(dtype=7)), None) == -2
    assert lib.fxb_tree_attn(None, None) == -1


def kv_args(**kw):
    from fxb200 import _lib
    a = _lib.KvArgs()
    a.elem_size, a.L, a.P, a.H, a.page, a.D, a.S, a.W = 2, 2, 8, 2, 16, 64, 2, 4
    a.k = a.v = a.table = a.n_pages = a.lens = a.ref = 256
    a.table_ss = 4
    for n in ("k", "v"):
        for s in ("sl", "sp", "sh", "st"):
            setattr(a, f"{n}_{s}", 64)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(page=20), "page 20"), (dict(S=0), "S=0"), (dict(S=5000), "S=5000"), (dict(W=0), "W=0"), (dict(P=0), "P=0"),
    (dict(table=0), "NULL"), (dict(table_ss=3), "row stride"), (dict(elem_size=1), "elem_size"), (dict(D=12), "D=12"),
    (dict(L=0), "L=0"), (dict(k=8), "aligned"), (dict(k_st=4), "strides"), (dict(v_sp=-64), "strides")])
def test_kv_calls_refuse(lib, change, word):
    a = kv_args(**change)
    p = ctypes.c_void_p(512)
    assert lib.fxb_kv_commit(ctypes.byref(a), p, 4, 4, p, None, p, None) == -1
    assert word in err()
    assert lib.fxb_kv_fork(ctypes.byref(a), p, p, None) == -1
    assert word in err()


def test_kv_calls_refuse_their_own_arguments(lib):
    p, a = ctypes.c_void_p(512), kv_args()
    assert lib.fxb_kv_commit(ctypes.byref(a), p, 4, 4, p, None, ctypes.c_void_p(256), None) == -1  # lens_out is lens
    assert "lens_out" in err()
    assert lib.fxb_kv_commit(ctypes.byref(a), p, 65, 65, p, None, p, None) == -1 and "T=65" in err()
    assert lib.fxb_kv_commit(ctypes.byref(a), p, 4, 4, None, None, p, None) == -1
    assert lib.fxb_kv_fork(ctypes.byref(a), None, p, None) == -1
    assert lib.fxb_kv_fork(ctypes.byref(a), p, ctypes.c_void_p(8), None) == -1
    assert lib.fxb_kv_commit(None, p, 4, 4, p, None, p, None) == -1
    assert lib.fxb_kv_fork_workspace(0, 3) == 0


def test_verify_refuses(lib):
    p = ctypes.c_void_p(256)

    def call(B=1, T=2, V=8, tokens=p, q=None, p_st=8, q_st=8):
        return lib.fxb_verify_tree(tokens, p, p, p, 16, p_st, q, 16, q_st, p, p, p, p, B, T, V, None)

    for kw in (dict(B=0), dict(T=65), dict(T=0), dict(V=0), dict(tokens=None), dict(p_st=-1), dict(q=p, q_st=-1)):
        assert call(**kw) == -1 and "fxb_verify_tree" in err()


def test_wrappers_refuse_on_the_host():
    from fxlm import kv_commit, kv_fork, kv_reserve, tree_attention, verify_tree
    bf = torch.bfloat16
    q = torch.zeros(1, 2, 4, 64, dtype=bf)
    kv = torch.zeros(1, 2, 2, 64, dtype=bf)
    pages = torch.zeros(4, 2, 16, 64, dtype=bf)
    i = torch.zeros(1, dtype=torch.int32)
    rest = (i[:, None], i, i, torch.zeros(1, 2, dtype=torch.int64))
    with pytest.raises(TypeError, match="cuda"):
        tree_attention(q, kv, kv, pages, pages, *rest)
    with pytest.raises(TypeError, match="share"):
        tree_attention(q, kv.float(), kv, pages, pages, *rest)
    with pytest.raises(TypeError, match="share"):
        tree_attention(q.double(), kv.double(), kv.double(), pages.double(), pages.double(), *rest)
    with pytest.raises(ValueError, match="head_dim 32"):
        tree_attention(q[..., :32], kv[..., :32], kv[..., :32], pages[..., :32], pages[..., :32], *rest)
    with pytest.raises(ValueError, match="shape mismatch"):
        tree_attention(q[:, :, :3], kv, kv, pages, pages, *rest)
    with pytest.raises(ValueError, match="T=65"):
        z = torch.zeros(1, 65, 2, 64, dtype=bf)
        tree_attention(z, z, z, pages, pages, *rest)
    with pytest.raises(ValueError, match="pages"):
        tree_attention(q, kv, kv, pages, pages[:2], *rest)
    with pytest.raises(ValueError):
        tree_attention(q[0], kv, kv, pages, pages, *rest)
    p = torch.zeros(1, 2, 8)
    with pytest.raises(TypeError, match="cuda"):
        verify_tree(torch.zeros(1, 2, dtype=torch.int64), i, i, p, p[..., 0])
    with pytest.raises(ValueError, match="T=65"):
        verify_tree(torch.zeros(1, 65, dtype=torch.int64), i, i, p, p[..., 0])
    with pytest.raises(ValueError):
        verify_tree(torch.zeros(2, dtype=torch.int64), i, i, p, p[..., 0])
    pool = torch.zeros(2, 4, 2, 16, 64, dtype=bf)
    args = (i[:, None], i, i, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError, match="cuda"):
        kv_commit(pool, pool, *args, i[:, None], i)
    with pytest.raises(TypeError, match="cuda"):
        kv_fork(pool, pool, *args, i)
    with pytest.raises(TypeError, match="cuda"):
        kv_reserve(*args, i, 16)


def test_tree_masks():
    from fxlm import tree_masks
    par = torch.tensor([[-1, 0, 0, 1, 3], [-1, 0, 1, 2, 3]], dtype=torch.int32)
    assert tree_masks(par).tolist() == [[1, 3, 5, 11, 27], [1, 3, 7, 15, 31]]
    chain = torch.arange(-1, 63, dtype=torch.int32)[None]
    assert tree_masks(chain)[0, -1].item() == -1 and tree_masks(chain)[0, 62].item() == 2 ** 63 - 1
    with pytest.raises(ValueError):
        tree_masks(torch.zeros(1, 65, dtype=torch.int32))


def test_tree_batch_and_masks_agree():
    from fxlm import tree_masks
    from fxlm.decode import tree_batch
    trees = [([5, 6, 7, 8], [-1, 0, 0, 2]), ([], []), (list(range(64)), list(range(-1, 63)))]
    tok, par, n, mask, depth = tree_batch(trees, "cpu")
    assert n.tolist() == [4, 0, 64] and tok[0].tolist()[:5] == [5, 6, 7, 8, 0]
    want = tree_masks(par)
    assert mask[0, :4].tolist() == want[0, :4].tolist() and mask[2].tolist() == want[2].tolist()
    assert depth[0, :4].tolist() == [0, 1, 1, 2] and depth[2].tolist() == list(range(64))


def test_draft_from_text():
    from fxlm.decode import draft_from_text
    # the last three tokens occurred twice: both continuations, common beginning merged
    seq = [1, 2, 3, 9, 8, 7, 1, 2, 3, 9, 5, 1, 2, 3]
    tok, par = draft_from_text(seq, 7)
    assert tok[0] == 3 and tok.count(9) == 1 and par[0] == -1 and all(0 <= p < c for c, p in enumerate(par) if c)
    paths = set()
    for c in range(len(tok)):
        p, x = [], c
        while x > 0:
            p.insert(0, tok[x])
            x = par[x]
        paths.add(tuple(p))
    assert (9, 5, 1) in paths and (9, 8, 7) in paths
    assert draft_from_text([4], 5) == ([4], [-1])
    assert draft_from_text([4, 5, 6], 5) == ([6], [-1])          # nothing to repeat
    assert draft_from_text(seq, 1) == ([3], [-1])
    assert len(draft_from_text([7] * 200, 64)[0]) <= 64


def test_next_probs():
    from fxlm.decode import next_probs
    x = torch.tensor([[1.0, 3.0, 3.0, 2.0, -1.0]])
    p = next_probs(x, 0.5, 2)
    assert p[0, 1] == p[0, 2] == 0.5 and p[0, 0] == p[0, 3] == p[0, 4] == 0
    assert torch.allclose(next_probs(x, 1.0, 0), torch.softmax(x, -1))


def test_wrappers_take_tensors_and_say_what_is_wrong():
    from fxlm import kv_commit, kv_fork, kv_reserve, verify_tree
    i = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(2, 4, 2, 16, 64, dtype=torch.bfloat16)
    args = (i[:, None], i, i, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(AttributeError):
        kv_commit(pool, pool, None, i, i, i, i[:, None], i)
    with pytest.raises(TypeError, match="page_table"):
        kv_commit(pool, pool, i.long()[:, None], *args[1:], i[:, None], i)
    with pytest.raises(TypeError, match="page_table"):
        kv_fork(pool, pool, *args, [0])
    with pytest.raises(TypeError):
        kv_reserve(*args, i, "16")
    with pytest.raises(TypeError, match="int64"):
        verify_tree(torch.zeros(1, 2), i, i, torch.zeros(1, 2, 8), torch.zeros(1, 2))


class _Buffer:
    """Stands in for a tensor of the allocator and records its memsets."""

    def __init__(self, n, log):
        self.n, self.log = n, log
        log.append(("new", self))

    def numel(self):
        return self.n

    def __getitem__(self, part):
        return self

    def zero_(self):
        self.log.append(("zero", self))


@pytest.fixture
def allocations(monkeypatch):
    from fxb200 import ops
    log = []
    monkeypatch.setattr(torch, "empty", lambda n, **kw: _Buffer(n, log))
    monkeypatch.setattr(ops, "_STREAM_WS", {})
    return log


def test_workspaces_of_plain_captures_are_their_own(monkeypatch, allocations):
    # plain captures share one capture stream: each call's buffer is new and zeroed in its own graph, and none
    # of them is handed to another call or kept where a larger request could drop it
    from fxb200 import ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    eager = ops.stream_workspace("k", 0, 7, 100, 16)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    first = ops.stream_workspace("k", 0, 7, 100, 16)
    second = ops.stream_workspace("k", 0, 7, 100, 16)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert len({id(x) for x in (eager, first, second)}) == 3
    assert [x for what, x in allocations if what == "zero"] == [eager, first, second]
    assert ops.stream_workspace("k", 0, 7, 50, 16) is eager
    assert list(ops._STREAM_WS.values()) == [eager]


def test_workspaces_of_a_table_are_kept(monkeypatch, allocations):
    from fxb200 import ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    table = {}
    with ops.graph_workspaces(table):
        ws = ops.stream_workspace("k", 0, 7, 100, 16)
        assert ops.stream_workspace("k", 0, 7, 100, 16) is ws and list(table.values()) == [ws]
    assert not ops._STREAM_WS


def test_gemm_workspaces_of_plain_captures_are_their_own(monkeypatch, allocations):
    from fxb200 import ops

    class Stream:
        cuda_stream = 7

    monkeypatch.setattr(ops, "_GEMM_WS", {})
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    device = torch.device("cuda", 0)
    first, second = ops._gemm_workspace(device), ops._gemm_workspace(device)
    assert first is not second and not ops._GEMM_WS
    assert [x for what, x in allocations if what == "zero"] == [first, second]
    with ops.graph_workspaces({}):
        assert ops._gemm_workspace(device) is ops._gemm_workspace(device)


def test_commit_refuses_lengths_written_over_its_arguments(lib):
    a = kv_args()
    a.n_pages, a.ref, a.table = 1024, 2048, 4096
    path, n_path, room = (ctypes.c_void_p(x) for x in (512, 768, 8192))
    for out in (256, 1024, 2048, 4096, 512, 768, 8192):
        assert lib.fxb_kv_commit(ctypes.byref(a), path, 4, 4, n_path, room, ctypes.c_void_p(out), None) == -1
        assert "lens_out" in err()
    assert lib.fxb_kv_commit(ctypes.byref(a), path, 4, 4, n_path, room, None, None) == -1 and "lens_out" in err()


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_arguments_on_several_devices_are_refused():
    # tensors without storage stand in for those of two GPUs: one argument on the other GPU at a time
    from torch._subclasses.fake_tensor import FakeTensorMode
    from fxlm import kv_commit, kv_fork, kv_reserve, tree_attention, verify_tree
    bf, i32, i64, f32 = torch.bfloat16, torch.int32, torch.int64, torch.float32

    def refused(fn, shapes, **kw):
        for odd in shapes:
            args = {n: torch.empty(*s, dtype=d, device="cuda:1" if n == odd else "cuda:0") for n, (s, d) in shapes.items()}
            with pytest.raises(ValueError, match="cuda:1"):
                fn(**args, **kw)

    cache = dict(page_table=((1, 4), i32), n_pages=((1,), i32), lens=((1,), i32), ref=((4,), i32))
    pools = dict(k=((2, 4, 2, 16, 64), bf), v=((2, 4, 2, 16, 64), bf))
    with FakeTensorMode():
        refused(tree_attention, dict(
            q=((1, 2, 4, 64), bf), k=((1, 2, 2, 64), bf), v=((1, 2, 2, 64), bf), k_pages=((4, 2, 16, 64), bf),
            v_pages=((4, 2, 16, 64), bf), page_table=((1, 4), i32), ctx_lens=((1,), i32), n_nodes=((1,), i32),
            tree_mask=((1, 2), i64), out=((1, 2, 4, 64), bf)))
        refused(verify_tree, dict(
            tokens=((1, 2), i64), parents=((1, 2), i32), n_nodes=((1,), i32), target_probs=((1, 2, 8), f32),
            u=((1, 2), f32), draft_probs=((1, 2, 8), f32)))
        refused(kv_commit, dict(**pools, **cache, path=((1, 2), i32), n_path=((1,), i32), room=((1,), i32), out=((1,), i32)))
        refused(kv_reserve, dict(**cache, room=((1,), i32)), page=16)
        refused(kv_fork, dict(**pools, **cache, parents=((1,), i32)))


def test_tree_attn_takes_one_mask_for_all_rows(lib):
    # (a row stride of 0 passes; the next check, of the workspace, stops the call here)
    assert lib.fxb_tree_attn(ctypes.byref(tree_args(B=3, mask_sb=0)), None) == -1 and "workspace" in err()
    for kw in (dict(mask_sb=-4), dict(table_sb=0)):
        assert lib.fxb_tree_attn(ctypes.byref(tree_args(B=3, **kw)), None) == -1 and "row stride" in err()


def test_strides_of_single_entries_may_be_anything(lib):
    odd = {f"{n}_{s}": 7 for n in ("q", "k", "v", "o") for s in ("sb", "st", "sh")}
    a = tree_args(T=1, Hq=1, Hkv=1, P=1, **odd, kp_sp=3, kp_sh=-5, vp_sp=9, vp_sh=1)
    assert lib.fxb_tree_attn(ctypes.byref(a), None) == -1 and "workspace" in err()
    p = ctypes.c_void_p(512)
    k = kv_args(L=1, P=1, H=1, k_sl=7, k_sp=3, k_sh=1, v_sl=-9, v_sp=5, v_sh=3)
    assert lib.fxb_kv_fork(ctypes.byref(k), p, ctypes.c_void_p(8), None) == -1 and "workspace" in err()


def test_tree_masks_of_parents_that_are_none():
    # forward, to itself, outside the tree: on the GPU an index outside would end the process's context
    from fxlm import tree_masks
    par = torch.tensor([[-1, 1, 3, 0, 2], [7, 0, -9, 2 ** 31 - 1, 3]], dtype=torch.int32)
    assert tree_masks(par).tolist() == [[1, 2, 4, 9, 20], [1, 3, 4, 8, 24]]


@pytest.fixture
def binding_build(monkeypatch, tmp_path):
    """fxb200.build with an empty lib folder and a compiler that only writes its output; the commands it was given."""
    import importlib
    import subprocess
    build = importlib.import_module("fxb200.build")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    return build, ran


def test_binding_is_rebuilt_for_another_torch(binding_build, monkeypatch):
    # a binding made for another version of torch has another ABI, however new its file is
    import importlib.metadata
    build, ran = binding_build
    build._build_binding()
    build._build_binding()
    assert len(ran) == 1
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "99.0")
    build._build_binding()
    build._build_binding()
    assert len(ran) == 2


def test_library_builds_without_torch(binding_build, monkeypatch, capsys):
    import importlib.util
    build, ran = binding_build
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    build._build_binding()
    assert not ran and "torch is not installed" in capsys.readouterr().err


def test_a_table_of_workspaces_serves_one_capture(monkeypatch, allocations):
    from fxb200 import ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    table = {}
    with ops.graph_workspaces(table):
        ops.stream_workspace("k", 0, 7, 100, 16)
    with pytest.raises(ValueError, match="another capture"):
        with ops.graph_workspaces(table):
            pass
    assert ops._CAPTURE_WS is None
