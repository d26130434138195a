"""GPU tests of generation with a KV cache: logits of token trees against the
model's own forward pass, and generate_cached against the sampler's loop."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


@pytest.fixture(autouse=True)
def _clean_error_word(dev):
    yield
    from fxb200 import _lib
    code = _lib.device_error(clear=True)
    assert code == 0, f"device error word {code}"


def model_of(dev, dtype, seq_len=96, n_head=2, d_model=128):
    from fxlm import GPT, GPTConfig
    torch.manual_seed(0)
    m = GPT(GPTConfig(vocab_size=256, seq_len=seq_len, n_layer=3, n_head=n_head, d_model=d_model))
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 2:
                p.mul_(3)
        m.pos_emb.normal_(std=0.3)
    return m.to(dev, dtype).eval()


# fp32: rounding of sums of up to 1024 products through 3 layers; 16 bits: the rounding of the activations
# (unit roundoffs 2^-8 and 2^-11, about ten roundings a layer, in quadrature)
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2), (torch.float16, 4e-3)])
def test_tree_logits_are_the_models(dev, dtype, tol):
    from fxlm.decode import PagedKVCache, tree_batch, tree_logits
    m = model_of(dev, dtype)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (1, 20, 71)]
    cache = PagedKVCache(3, 2, 64, 3, 160, dev, dtype, page=16)
    with torch.inference_mode():
        while any(len(s) - 1 > int(n) for s, n in zip(seqs, cache.lens)):  # the sequences but for their last tokens
            parts = [s[int(n):min(int(n) + 33, len(s) - 1)] for s, n in zip(seqs, cache.lens)]
            tok, par, n, mask, depth = tree_batch([(p, list(range(-1, len(p) - 1))) for p in parts], dev)
            cache.reserve(n)
            tree_logits(m, cache, tok, n, mask, depth)
            cache.commit((par + 1).contiguous(), n)
        trees = [(s[-1:] + [5, 6, 7, 8, 9], [-1, 0, 0, 1, 3, 2]) for s in seqs]
        tok, par, n, mask, depth = tree_batch(trees, dev)
        cache.reserve(n)
        got = tree_logits(m, cache, tok, n, mask, depth)
        for b, s in enumerate(seqs):
            for i in range(6):
                path, c = [], i
                while c > 0:
                    path.insert(0, trees[b][0][c])
                    c = trees[b][1][c]
                want = m(torch.tensor([s + path], device=dev))[0, -1].double()
                err = (got[b, i].double() - want).norm() / want.norm()
                assert err < tol, (b, i, float(err))
    cache.check()


@pytest.mark.parametrize("draft", [0, 1, 7, 20])
@pytest.mark.parametrize("prompt,new", [(1, 40), (30, 20), (70, 60), (96, 5), (120, 3)])
def test_generate_cached_is_generate(dev, draft, prompt, new):
    # top_k = 1 leaves one token: both loops have to find the same one (fp32), past the window too
    from fxlm import generate_cached
    from fxlm.sample import generate
    m = model_of(dev, torch.float32)
    ids = (torch.arange(prompt, device=dev) * 7) % 11
    want = generate(m, ids, new, temperature=1.0, top_k=1)
    stats = {}
    got = generate_cached(m, ids, new, temperature=1.0, top_k=1, draft=draft, samples=2, stats=stats)
    assert got.shape == (2, prompt + new)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[0])
    if draft == 0:
        assert stats["tokens"] == 2 * stats["steps"]


def test_drafts_are_accepted(dev):
    # drafts looked up in the text itself: some are right, and what they save are steps, not tokens
    from fxlm import generate_cached
    m = model_of(dev, torch.bfloat16, seq_len=512)
    stats = {}
    generate_cached(m, torch.tensor([1, 2, 3], device=dev), 300, temperature=1.0, top_k=1, draft=7, stats=stats)
    assert stats["tokens"] == 300
    assert stats["steps"] < 300


def test_samples_differ_and_repeat_with_the_seed(dev):
    from fxlm import generate_cached
    m = model_of(dev, torch.bfloat16)
    ids = torch.tensor([3, 1, 4], device=dev)

    def go():
        g = torch.Generator(device=dev).manual_seed(7)
        return generate_cached(m, ids, 30, temperature=1.0, top_k=0, generator=g, draft=5, samples=4)

    a, b = go(), go()
    assert torch.equal(a, b) and len({tuple(x) for x in a.tolist()}) == 4


def test_sample_command(dev, tmp_path):
    from dataclasses import asdict
    from fxlm import sample
    m = model_of(dev, torch.float32)
    torch.save({"config": asdict(m.cfg), "model": {k: v.float().cpu() for k, v in m.state_dict().items()},
                "meta": {"tokenizer": "bytes"}, "args": {"dtype": "fp32"}}, tmp_path / "c.pt")
    args = ["--ckpt", str(tmp_path / "c.pt"), "--prompt", "ab", "--max-new", "12", "--top-k", "1"]
    assert sample.main(args) == sample.main(args + ["--draft", "4"])
    two = sample.main(args + ["--draft", "4", "--num-samples", "2"])
    assert two == "\n".join([sample.main(args)] * 2)


def test_logits_without_probabilities_raise(dev):
    from fxlm import generate_cached
    m = model_of(dev, torch.float32)
    with torch.no_grad():
        m.lnf_w.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="probabilit"):
        generate_cached(m, torch.tensor([3, 1, 4], device=dev), 6, draft=2, samples=2)


def test_gradients_are_not_cut_silently(dev):
    # a decoding step works with gradients enabled; logits that would carry a graph without attention are refused
    from fxlm.decode import DecodeStep, PagedKVCache, tree_batch, tree_logits
    m = model_of(dev, torch.float32)
    cache = PagedKVCache(3, 2, 64, 1, 160, dev, torch.float32)
    tok, par, n, mask, depth = tree_batch([([1, 2], [-1, 0])], dev)
    cache.reserve(n)
    with pytest.raises(ValueError, match="no_grad"):
        tree_logits(m, cache, tok, n, mask, depth)
    step = DecodeStep(m, cache, 2, 1.0, 1)
    for _ in range(4):
        (path, nxt), = step([([1], [-1])], torch.zeros(1, 2, device=dev))
        assert path == [0] and nxt >= 0
    cache.check()


@pytest.mark.parametrize("draft", [0, 1, 5])
def test_generated_tokens_follow_the_model(dev, draft):
    # the first three tokens of many samples, each continuation's count within 5 standard deviations of what the
    # model gives it when the window is run again for every token, as the sampler's loop does. The prompt is
    # chosen so that what is drafted from it is one of the tokens that can follow
    from fxlm import generate_cached
    from fxlm.decode import draft_from_text, next_probs
    m, S, K = model_of(dev, torch.float32), 4000, 3
    with torch.inference_mode():
        tries = torch.tensor([[5, 6, t, 9, 8, 5, 6] for t in range(256)], device=dev)
        p = next_probs(m(tries)[:, -1], 1.0, K)
        t = int(p[torch.arange(256), torch.arange(256)].argmax())
        assert 0.1 < float(p[t, t]) < 0.9
        prompt = tries[t]
        paths, prob = prompt[None], torch.ones(1, dtype=torch.float64, device=dev)
        for _ in range(3):
            top = next_probs(m(paths)[:, -1], 1.0, K).double().topk(K, -1)
            paths = torch.cat([paths.repeat_interleave(K, 0), top.indices.reshape(-1, 1)], 1)
            prob = (prob[:, None] * top.values).reshape(-1)
    if draft:
        assert draft_from_text(prompt.tolist(), draft + 1)[0][1] == t
    g = torch.Generator(device=dev).manual_seed(2)
    out = generate_cached(m, prompt, 3, temperature=1.0, top_k=K, generator=g, draft=draft, samples=S)
    hits = (out[:, None] == paths[None]).all(-1).double().sum(0)
    assert int(hits.sum()) == S
    assert ((hits - S * prob).abs() <= 5 * (S * prob * (1 - prob)).sqrt() + 1).all()
