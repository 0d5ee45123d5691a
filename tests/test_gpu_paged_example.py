"""The paged decoding example: steps over the cache against one pass over the whole texts (GPU)."""

import importlib.util
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("paged_decode", ROOT / "examples" / "paged_decode.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["paged_decode"] = mod
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("cache", ["int8", "bfloat16", "float16"])
def test_steps_agree_with_one_pass(example, pkg, cache):
    """Every step's log probabilities are those of one ragged pass over prompts and answers: the
    same rows with the same stored keys and values, so only the order of the attention's sums
    differs. Where that moves an INT8 activation by a step, a logit (of size 1) moves by less
    than 1/127 a layer and projection; 0.1 bounds them all."""
    dt = getattr(torch, cache)
    model = example.Decoder(pkg)
    prompts = [[1, 5, 9, 2], [7] * 33, [3], list(range(100, 117))]
    answers, caches, pages = example.generate(model, prompts, 9, dt)
    texts = [p + [t["id"] for t in a][:-1] for p, a in zip(prompts, answers)]
    fresh = [pkg.PagedKVCache(c.num_pages, c.page_size, c.kv_heads, c.head_dim, dt) for c in caches]
    table = torch.from_numpy(pages.table).cuda()
    rows = [(t, s, i) for s, text in enumerate(texts) for i, t in enumerate(text)]
    tok, seq, pos = (example.int32(c) for c in zip(*rows))
    r = pkg.token_logprobs(model.step(fresh, table, tok, seq, pos), top_k=3)
    first = 0
    for prompt, text, answer in zip(prompts, texts, answers):
        for i, t in enumerate(answer):
            row = first + len(prompt) - 1 + i
            got = dict(zip(r.top_ids[row].tolist(), r.top_logprobs[row].tolist()))
            assert abs(got.get(t["id"], -1e9) - t["logprob"]) <= 0.1
            assert abs(float(r.entropy[row]) - t["entropy"]) <= 0.1
        first += len(text)
    for a, b in zip(caches, fresh):
        # the stored rows are the same but for such steps
        ka, va = a.read(table, seq, pos)
        kb, vb = b.read(table, seq, pos)
        assert (ka - kb).abs().max() <= 0.1 and (va - vb).abs().max() <= 0.1


def test_command_line(example, capsys, monkeypatch):
    monkeypatch.setattr(sys, "argv", ["paged_decode.py", "--tokens", "3", "--cache", "bfloat16"])
    example.main()
    out = capsys.readouterr().out
    assert out.count("prompt of") == 4 and out.count("logprob") == 12
