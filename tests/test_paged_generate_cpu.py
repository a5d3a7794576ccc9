"""Generation from a cache in pages on the host: the same tokens as from the rectangular cache, with and without drafts; pages come back."""
import pytest
import torch

from llmc_b200.models import generate as G
from llmc_b200.models import llama3
from llmc_b200.models import paged as P
from llmc_b200.ops import kernels as KN

DESC = "llama3:l=2,c=64,h=4,kv=2,t=48,v=97,m=32,f=1.0"
PROMPTS = [[5, 9, 5, 9, 5], [3], list(range(40, 59)), [8, 8]]


def small_model(desc=DESC, seed=7):
    m = llama3.Llama(llama3.config_from_descriptor(desc), "cpu", torch.float32, recompute=0)
    m.init_random(seed)
    for n in ("qkvw", "attprojw", "fc12w", "fcprojw", "lmhead"):
        m.params[n].mul_(4.0)
    return m


@pytest.mark.parametrize("drafts", [0, 1, 5, 12])
@pytest.mark.parametrize("desc", [DESC, "llama3:l=1,c=64,h=4,kv=1,t=48,v=13,m=16,f=1.3"])
def test_greedy_tokens_are_those_of_the_rectangular_cache(desc, drafts):
    m = small_model(desc)
    prompts = [[t % m.cfg.vocab_size for t in p] for p in PROMPTS]
    want = G.generate(m, prompts, 20, temperature=0.0)
    assert P.generate_paged(m, prompts, 20, temperature=0.0, drafts=drafts, rows=8) == want
    stop = want[0][7]
    assert P.generate_paged(m, prompts, 20, temperature=0.0, drafts=drafts, rows=8, stop_tokens=(stop,), echo=True) == G.generate(m, prompts, 20, temperature=0.0, stop_tokens=(stop,), echo=True) \
        or stop in sum(prompts, [])                     # (a prompt that holds it is cut by the one and not by the other)


def test_the_context_ends_a_sequence():
    m = small_model()
    got = P.generate_paged(m, [list(range(30)), [1]], 100, temperature=0.0, drafts=6, rows=8)
    assert [len(g) for g in got] == [18, 47]
    assert got == P.generate_paged(m, [list(range(30)), [1]], 100, temperature=0.0, rows=16)
    assert P.generate_paged(m, [list(range(48))], 5) == [[]]


def test_drafts_are_checked_and_kept(monkeypatch):
    """A model that counts in a circle: the drafts looked up in the text are right, and several tokens a step are kept."""
    m = small_model()
    steps = []
    forward = P.PagedDecoder.forward

    def counting(self, sequences, tokens, parents=None, every=False):
        logits = forward(self, sequences, tokens, parents, every)
        steps.append(sum(len(t) for t in tokens))
        # the next of 0 .. 6, whatever the model says
        flat = [t for l in tokens for t in (l if every else l[-1:])]
        return torch.nn.functional.one_hot(torch.tensor([(t + 1) % 7 for t in flat]), m.cfg.vocab_size).float()

    monkeypatch.setattr(P.PagedDecoder, "forward", counting)
    got = P.generate_paged(m, [[0, 1, 2, 3, 4, 5, 6, 0, 1], [2]], 25, temperature=0.0, drafts=8, rows=8)
    assert got == [[(2 + i) % 7 for i in range(25)], [(3 + i) % 7 for i in range(25)]]
    assert len(steps) < 20


def test_sampling_with_drafts_runs():
    m = small_model()
    got = P.generate_paged(m, PROMPTS, 12, temperature=0.9, top_p=0.8, drafts=7, generator=torch.Generator().manual_seed(1), rows=8)
    assert [len(g) for g in got] == [12] * 4


def test_logits_of_steps_of_any_form():
    m = small_model()
    g = torch.Generator().manual_seed(0)
    tok = torch.randint(0, m.cfg.vocab_size, (2, 24), generator=g, dtype=torch.int32)
    m.forward(tok)
    full = m.logits()[..., :m.cfg.vocab_size].clone()
    near = lambda a, b: torch.allclose(a, b, atol=1e-4, rtol=1e-4)
    d = P.PagedDecoder(m, 12, 8)
    a, b = d.open(), d.open()
    assert near(d.forward([a], [tok[0, :5].tolist()]), full[:1, 4])
    got = d.forward([b, a], [tok[1, :11].tolist(), tok[0, 5:6].tolist()])
    assert near(got, torch.stack([full[1, 10], full[0, 5]]))
    got = d.forward([a, b], [tok[0, 6:9].tolist(), tok[1, 11:12].tolist()], every=True)
    assert near(got, torch.cat([full[0, 6:9], full[1, 11:12]]))
    # a tree whose right branch is 0, 2, 3; the others are not kept
    t = tok[0, 9:12].tolist()
    got = d.forward([a], [[t[0], 1, t[1], t[2], 4]], [[-1, 0, 0, 2, -1]], every=True)
    assert near(got[[0, 2, 3]], full[0, 9:12])
    d.keep([a], [5], [[0, 2, 3]])
    assert a.length == 12 and near(d.forward([a], [tok[0, 12:20].tolist()], every=True), full[0, 12:20])
    used = len(a.pages) + len(b.pages)
    assert used + len(d.free) == 12
    d.close(a), d.close(b)
    assert sorted(d.free) == list(range(12))


def test_refusals():
    m = small_model()
    d = P.PagedDecoder(m, 2, 8)
    s = d.open()
    for sequences, tokens, parents in (([s], [[]], None), ([], [], None), ([s, s], [[1], [1]], None), ([s], [[1, 2]], [[-1]]), ([s], [[1] * 49], None), ([s], [[1, 2]], [[-1, 1]])):
        with pytest.raises(ValueError):
            d.forward(sequences, tokens, parents)
    d.close(s)
    with pytest.raises(RuntimeError):
        d.forward([s], [[1] * 17])
    d.forward([s], [[1, 2, 3]])
    for kept in ([2, 1], [0, 0], [3], [-1]):
        with pytest.raises(ValueError):
            d.keep([s], [3], [kept])
    for bad in ([], [[]], [[1] * 49]):
        with pytest.raises(ValueError):
            P.generate_paged(m, bad, 3)
    for drafts in (-1, 64):
        with pytest.raises(ValueError):
            P.generate_paged(m, [[1]], 3, drafts=drafts)


def test_drafted_tree():
    assert P.drafted_tree([4, 1, 2, 9, 1, 2], 6) == ([2, 9, 1, 2], [-1, 0, 1, 2])
    tree, parents = P.drafted_tree([1, 2, 3, 4, 1, 2, 3, 5, 1, 2], 8)
    assert tree[0] == 2 and tree[1] == 3 and len(tree) == len(parents) <= 9
    assert len({(p, t) for p, t in zip(parents, tree)}) == len(tree)          # no child twice
    assert P.drafted_tree([1], 5) == ([1], [-1]) and P.drafted_tree([1, 1, 1], 0) == ([1], [-1])
    for n in range(2, 40):
        tree, parents = P.drafted_tree([i * i % 7 for i in range(n)], n % 9)
        assert len(tree) <= n % 9 + 1 and all(-1 <= p < i for i, p in enumerate(parents)) and parents[1:].count(-1) == 0


def test_command_line(tmp_path):
    import train_llama3
    args = train_llama3.build_parser().parse_args(["--prompt_tokens", "5,9,5,9,5;3", "--max_gen_len", "9", "--temperature", "0", "--page_rows", "8", "--drafts", "4"])
    m = small_model()
    assert train_llama3.generate_from_args(m, args) == G.generate(m, [[5, 9, 5, 9, 5], [3]], 9, temperature=0.0)
    for wrong in (["--drafts", "4"], ["--page_rows", "12"], ["--page_rows", "8", "--drafts", "64"], ["--page_rows", "8", "--use_kv", "0"]):
        with pytest.raises(SystemExit):
            train_llama3.generate_from_args(m, train_llama3.build_parser().parse_args(["--prompt_tokens", "1"] + wrong))
    assert KN.launch_count() >= 0
