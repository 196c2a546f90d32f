"""The engine between two steps: caches that keep attention weights, their eviction, generation with drafted tokens, and all
of it together."""
import pytest
import torch

from conftest import CONFIGS, TINY_D
from helpers import tokens

pytestmark = pytest.mark.gpu

ONE_LAYER = {**TINY_D, "num_hidden_layers": 1}
# head size 128, one layer, longer positions
ONE_WIDE = {**ONE_LAYER, "head_dim": 128, "num_attention_heads": 8, "num_key_value_heads": 2, "max_position_embeddings": 8192,
            "rope_scaling": None}


def _model(config, dtype, seed=3):
    import camelid_b200
    return camelid_b200.from_random(config, seed=seed, dtype=dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["tiny_b", "tiny_d"])
def test_tracked_cache_gives_the_same_logits_and_whole_weights(cuda, model_folders, dtype, name):
    """Weights of a row sum to one: after a prompt of n tokens (the last 32 are observed when it is longer than 8) and t single or
    drafted tokens, a kv head's scores of a sequence sum to (heads / kv heads) * (observed + t)."""
    import camelid_b200
    lm = camelid_b200.load(model_folders[name], dtype=dtype)
    cfg = CONFIGS[name]
    group = cfg["num_attention_heads"] // cfg["num_key_value_heads"]
    plain, tracked = lm.new_cache(1024), lm.new_cache(1024, track_weights=True)
    prompts = [tokens(i, n, cfg["vocab_size"]) for i, n in enumerate([70, 5, 33, 1])]
    slots = [[c.alloc_slot() for _ in prompts] for c in (plain, tracked)]
    # (a float32 step adds its products in an order of its own: the caches agree to rounding)
    limit = 2e-5 if dtype == "float32" else 4e-2

    def both(per_seq):
        out = [lm.step(c, [camelid_b200.StepEntry(s, t, list(range(len(t)))[-2:]) for s, t in zip(sl, per_seq)]) for c, sl in
               ((plain, slots[0]), (tracked, slots[1]))]
        assert float((out[0] - out[1]).abs().max()) <= limit * float(out[0].abs().max())
    both(prompts)
    seen = [min(len(p), 32) for p in prompts]
    for step in range(4):
        both([[step + 1]] * 4)
    both([[3, 4, 5], [6], [7, 8], [9]])
    seen = [s + 4 + n for s, n in zip(seen, (3, 1, 2, 1))]
    torch.cuda.synchronize()
    lengths = [tracked.length(s) for s in slots[1]]
    for i, s in enumerate(slots[1]):
        pages = tracked.book.pages[0][s]
        for e in range(cfg["num_hidden_layers"]):
            line = torch.cat([tracked.scores[0][e, p].cpu().double() for p in pages], dim=1)[:, :lengths[i]]
            assert bool((line >= 0).all())
            assert torch.allclose(line.sum(1), torch.full((cfg["num_key_value_heads"],), float(group * seen[i]), dtype=torch.float64), rtol=1e-5)


def test_captured_steps_add_their_weights_once(cuda, model_folders):
    """Captures run a step twice (warm-up) or once beside it; replayed steps of any length land in the same scores as eager ones."""
    import camelid_b200
    from camelid_b200 import KernelOptions
    group = 3
    results = []
    for options in (None, KernelOptions(capture_repeated_steps=False)):
        lm = camelid_b200.load(model_folders["tiny_d"], dtype="float32", options=options)
        if options is not None:
            lm.model.use_graphs = False
        cache = lm.new_cache(2048, track_weights=True)
        a, b = cache.alloc_slot(), cache.alloc_slot()
        sums = 0
        for n in (40, 40, 40, 5, 5, 5, 1, 1, 1):            # layouts that come back are captured
            lm.step(cache, [camelid_b200.StepEntry(s, tokens(n + s, n, 331), [n - 1]) for s in (a, b)])
            sums += min(n, 32) if n > 8 else n
        line = torch.cat([cache.scores[0][1, p] for p in cache.book.pages[0][b]], dim=1)[:, :cache.length(b)].double()
        assert torch.allclose(line.sum(1), torch.full_like(line.sum(1), float(group * sums)), rtol=1e-5)
        results.append(line)
        if options is None:
            toks = lm.model.decode_fed(cache, [a, b], [1, 2], 20)
            line = torch.cat([cache.scores[0][1, p] for p in cache.book.pages[0][b]], dim=1)[:, :cache.length(b)].double()
            assert toks.shape == (20, 2) and torch.allclose(line.sum(1), torch.full_like(line.sum(1), float(group * (sums + 20))), rtol=1e-5)
    assert torch.allclose(results[0], results[1], rtol=1e-3, atol=1e-4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("config", [ONE_LAYER, ONE_WIDE])
def test_evicted_sequence_goes_on_as_the_shorter_one(cuda, dtype, config):
    """With one layer a key depends on its token and position alone. Where the first and last positions are all that stays, the
    sequence must go on as a fresh one of those tokens: keys, values and logits, for several sequences and evictions."""
    import camelid_b200
    lm = _model(config, dtype)
    cache = lm.new_cache(4096, track_weights=True)
    vocab = config["vocab_size"]
    text = [tokens(10 + i, n, vocab) for i, n in enumerate([300, 64, 700, 130])]
    slots = [cache.alloc_slot() for _ in text]
    lm.step(cache, [camelid_b200.StepEntry(s, t, []) for s, t in zip(slots, text)])
    held = [list(t) for t in text]
    for keep in (129, 100, 64, 65, 7):
        # nothing of the middle stays: the first three and the last keep - 3
        assert lm.evict(cache, slots, keep, first=3, recent=keep - 3) == [min(len(h), keep) for h in held]
        held = [h if len(h) <= keep else h[:3] + h[len(h) - (keep - 3):] for h in held]
        cache.book.audit()
        new = [tokens(keep + i, 2, vocab) for i in range(len(held))]
        got = lm.step(cache, [camelid_b200.StepEntry(s, [t[0]], [0]) for s, t in zip(slots, new)])
        held = [h + [t[0]] for h, t in zip(held, new)]
        fresh = lm.new_cache(4096)
        other = [fresh.alloc_slot() for _ in held]
        want = lm.step(fresh, [camelid_b200.StepEntry(s, h, [len(h) - 1]) for s, h in zip(other, held)])
        limit = 3e-5 if dtype == "float32" else 4e-2
        assert float((got - want).abs().max()) <= limit * float(want.abs().max()), keep
        for i, (s, o) in enumerate(zip(slots, other)):
            for mine, theirs in ((cache.k[0], fresh.k[0]), (cache.v[0], fresh.v[0])):
                m = torch.cat([mine[0, p] for p in cache.book.pages[0][s]], dim=1)[:, :len(held[i])].float()
                t = torch.cat([theirs[0, p] for p in fresh.book.pages[0][o]], dim=1)[:, :len(held[i])].float()
                # a key turned several times is rounded each time: half a step a turn, of either of a pair's numbers
                steps = 5 * 2 * (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -19)
                assert float((m - t).abs().max()) <= steps * float(t.abs().max()), (keep, i)


def test_evict_chooses_by_the_kept_weights(cuda):
    """Each layer and kv head keeps the positions its own scores name; a sequence within its budget stays as it is."""
    import camelid_b200
    import plain_between as pb
    config = {**TINY_D, "num_hidden_layers": 2}
    lm = _model(config, "float32")
    cache = lm.new_cache(1024, track_weights=True)
    text = [tokens(i, n, 331) for i, n in enumerate([200, 90, 300])]
    slots = [cache.alloc_slot() for _ in text]
    lm.step(cache, [camelid_b200.StepEntry(s, t, []) for s, t in zip(slots, text)])
    lines = [torch.cat([cache.scores[0][:, p] for p in cache.book.pages[0][s]], dim=2).cpu() for s in slots]
    values = [torch.cat([cache.v[0][:, p] for p in cache.book.pages[0][s]], dim=2).cpu() for s in slots]
    assert lm.evict(cache, slots[::-1], 96, first=2, recent=20) == [96, 90, 96]
    for i, s in enumerate(slots):
        n = len(text[i])
        now = torch.cat([cache.v[0][:, p] for p in cache.book.pages[0][s]], dim=2).cpu()
        for e in range(2):
            for h in range(config["num_key_value_heads"]):
                places = pb.choose(lines[i][e, h].tolist(), n, 96, 2, 20) if n > 96 else list(range(n))
                assert torch.equal(now[e, h, :len(places)], values[i][e, h, places])
    cache.book.audit()
    assert cache.book.pools[0].n_held == 2 + 2 + 2


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafted_generation_gives_the_greedy_tokens(cuda, model_folders, dtype):
    import camelid_b200
    lm = camelid_b200.load(model_folders["tiny_d"], dtype=dtype)
    prompts = [tokens(80 + i, n, 331) for i, n in enumerate([30, 7, 64, 1])]
    want = lm.generate(prompts, max_tokens=40, stop_token_ids=())
    known = [list(p) + w for p, w in zip(prompts, want)]

    def right(history):
        full = next(k for k in known if k[:len(history)] == history)
        return full[len(history):len(history) + 5]

    def half(history):
        d = right(history)
        return [t if j % 3 != 2 else (t + 1) % 331 for j, t in enumerate(d)]
    if dtype == "bfloat16":                     # steps of other sizes round differently: near-ties may go the other way
        got = lm.generate(prompts, max_tokens=40, stop_token_ids=(), drafter=right)
        assert all(len(g) == 40 for g in got) and [g[0] for g in got] == [w[0] for w in want]
        return
    steps = {}
    for name, drafter in (("right", right), ("half", half), ("lookup", camelid_b200.PromptLookup(4, 2))):
        count = []
        assert lm.generate(prompts, max_tokens=40, stop_token_ids=(), drafter=drafter, on_step=lambda n: count.append(n)) == want, name
        steps[name] = len(count)
    assert steps["right"] <= 8 and steps["half"] <= 20
    stop = want[2][17]
    assert lm.generate(prompts, max_tokens=40, stop_token_ids=(stop,), drafter=half) == lm.generate(prompts, max_tokens=40, stop_token_ids=(stop,))


def test_drafted_sampling_is_the_requests_own(cuda, model_folders):
    """With a seed a request draws the same alone and in a batch; penalties count the drafts before a row; probabilities are taken."""
    import camelid_b200
    lm = camelid_b200.load(model_folders["tiny_b"], dtype="float32")
    prompts = [tokens(20 + i, n, 512) for i, n in enumerate([12, 5, 30])]
    look = camelid_b200.PromptLookup(3, 1)

    def certain(history):                       # a drafter that is sure of one token, as probabilities
        p = torch.full((2, 512), 0.0, device="cuda")
        p[:, history[-1]] = 1.0
        return [history[-1], history[-1]], p
    for options in ({"temperature": 0.9, "seed": 5}, {"temperature": 1.2, "top_p": 0.8, "seed": 6},
                    {"temperature": 0.7, "top_k": 20, "repeat_penalty": 1.3, "presence_penalty": 0.2, "seed": 7}):
        for drafter in (look, certain, lambda h: certain(h) if len(h) % 2 else look(h)):
            together = lm.generate(prompts, max_tokens=16, stop_token_ids=(), drafter=drafter, **options)
            alone = [lm.generate([p], max_tokens=16, stop_token_ids=(), drafter=drafter, **options)[0] for p in prompts]
            assert together == alone and all(len(t) == 16 for t in together)


def test_verification_of_no_sequences(cuda):
    from camelid_b200.sampling import Sampler, SamplingOptions
    for options in (SamplingOptions(), SamplingOptions(temperature=0.5, repeat_penalty=1.2, seed=1)):
        assert Sampler(options, 100, "cuda").verify(torch.zeros(0, 100, device=cuda), [], []) == ([], [])


def test_drafted_generation_over_a_cache_that_keeps_weights(cuda, model_folders):
    """Drafts that are always right: every row counts once, whatever steps brought it."""
    import camelid_b200
    lm = camelid_b200.load(model_folders["tiny_d"], dtype="float32")
    prompts = [tokens(60 + i, n, 331) for i, n in enumerate([30, 7, 12])]
    want = lm.generate(prompts, max_tokens=24, stop_token_ids=())
    known = [list(p) + w for p, w in zip(prompts, want)]

    def right(history):
        full = next(k for k in known if k[:len(history)] == history)
        return full[len(history):len(history) + 1 + len(history) % 4]
    cache = lm.new_cache(1024, track_weights=True)
    assert lm.generate(prompts, max_tokens=24, stop_token_ids=(), drafter=right, cache=cache) == want
    cache.book.audit()


def test_drafts_verification_and_eviction_together(cuda):
    """A long run as it would be served: prompts, steps with drafts, rejected ones rolled back, eviction over a budget; the captured
    single-token steps in between. With one layer and nothing of the middle kept, a fresh sequence of the positions that
    stayed says what the logits have to be."""
    import camelid_b200
    from camelid_b200.sampling import Sampler, SamplingOptions
    lm = _model(ONE_WIDE, "float32", seed=9)
    vocab = ONE_WIDE["vocab_size"]
    cache = lm.new_cache(2048, track_weights=True)
    sampler = Sampler(SamplingOptions(), vocab, "cuda")
    text = [tokens(i, n, vocab) for i, n in enumerate([150, 40])]
    slots = [cache.alloc_slot() for _ in text]
    lm.step(cache, [camelid_b200.StepEntry(s, t[:-1], []) for s, t in zip(slots, text)])
    held = [list(t[:-1]) for t in text]
    last = [t[-1] for t in text]
    for turn in range(12):
        drafts = [tokens(50 + turn + i, 3, vocab) if turn % 3 else [] for i in range(2)]
        fresh = lm.new_cache(2048)
        other = [fresh.alloc_slot() for _ in held]
        want = lm.step(fresh, [camelid_b200.StepEntry(s, h + [l] + d, list(range(len(h), len(h) + 1 + len(d)))) for s, h, l, d in
                               zip(other, held, last, drafts)])
        got = lm.step(cache, [camelid_b200.StepEntry(s, [l] + d, list(range(1 + len(d)))) for s, l, d in zip(slots, last, drafts)])
        assert float((got - want).abs().max()) <= 3e-5 * float(want.abs().max()), turn
        if drafts[0]:                           # the first draft of the first sequence is made right
            drafts[0][0] = int(got[0].argmax())
        counts, nexts = sampler.verify(got, drafts, [h + [l] for h, l in zip(held, last)])
        sampler.check()
        if drafts[0]:
            assert counts[0] == 1 or drafts[0][1] == int(got[1].argmax())
            counts = [0, min(counts[1], 0)]     # the step brought another token there: none of the drafts is in the cache as drafted
            nexts = [int(got[0].argmax()), int(got[4].argmax())]
        for i in range(2):
            cache.truncate(slots[i], cache.length(slots[i]) - (len(drafts[i]) - counts[i]))
            held[i] = held[i] + [last[i]] + drafts[i][:counts[i]]
            last[i] = int(nexts[i])
        if turn % 4 == 3:
            assert lm.evict(cache, slots, 60, first=2, recent=58) == [min(60, len(h)) for h in held]
            held = [h if len(h) <= 60 else h[:2] + h[len(h) - 58:] for h in held]
        cache.book.audit()
        assert [cache.length(s) for s in slots] == [len(h) for h in held]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_all_steps_of_a_tracked_cache_share_one_scratch(cuda, dtype):
    """Prompts, drafted steps and single tokens, eager and captured, of several layouts: the scratch is the one the cache was made with."""
    import camelid_b200
    lm = _model(ONE_WIDE, dtype)
    vocab = ONE_WIDE["vocab_size"]
    cache = lm.new_cache(2048, max_slots=4, track_weights=True)
    at = cache.weights_scratch.data_ptr()
    slots = [cache.alloc_slot() for _ in range(3)]
    for news in ([400, 30, 9], [1, 1, 1], [5, 1, 3], [5, 1, 3], [5, 1, 3], [8, 8, 8], [8, 8, 8], [20, 1, 40], [20, 1, 40], [1, 1, 1], [2, 1, 1]):
        lm.step(cache, [camelid_b200.StepEntry(s, tokens(n + s, n, vocab), [n - 1]) for s, n in zip(slots, news)])
    lm.model.decode_fed(cache, slots, [1, 2, 3], 5)
    lm.model.check_device_errors()
    spaces = [lm.model.workspace] + [g.ctx.ws for kept in (lm.model._graphs, lm.model._step_graphs) for g in kept[cache].values()]
    assert len(spaces) >= 4 and not any(name == "attn_weights" for ws in spaces for name, _ in ws._bufs)
    assert cache.weights_scratch.data_ptr() == at
    group = ONE_WIDE["num_attention_heads"] // ONE_WIDE["num_key_value_heads"]
    seen = [sum(min(n, 32) for n in each) + 5 for each in ((400, 1, 5, 5, 5, 8, 8, 20, 20, 1, 2), (30, 1, 1, 1, 1, 8, 8, 1, 1, 1, 1), (9, 1, 3, 3, 3, 8, 8, 40, 40, 1, 1))]
    for s, n in zip(slots, seen):
        line = torch.cat([cache.scores[0][0, p] for p in cache.book.pages[0][s]], dim=1)[:, :cache.length(s)].double()
        assert torch.allclose(line.sum(1), torch.full_like(line.sum(1), float(group * n)), rtol=1e-5)


def test_evicted_keys_whose_encoding_names_other_pairs(cuda):
    """A position encoding that calls its pairs neighbours in the mixer that always pairs split halves: evicted keys are a fresh sequence's."""
    import camelid_b200
    lm = _model(ONE_LAYER, "float32")
    lm.model.blocks[0].mixer.position.pairing = "interleaved"
    cache, fresh = lm.new_cache(512, track_weights=True), lm.new_cache(512)
    text = tokens(4, 200, ONE_LAYER["vocab_size"])
    slot, other = cache.alloc_slot(), fresh.alloc_slot()
    lm.step(cache, [camelid_b200.StepEntry(slot, text, [])])
    assert lm.evict(cache, [slot], 70, first=3, recent=67) == [70]
    lm.step(fresh, [camelid_b200.StepEntry(other, text[:3] + text[-67:], [])])
    m, t = (torch.cat([c.k[0][0, p] for p in c.book.pages[0][s]], dim=1)[:, :70] for c, s in ((cache, slot), (fresh, other)))
    # the rotary kernel rounds position * frequency: half a step of 2^-16 up to position 199, of 2^-17 up to 69; a pair is at most
    # sqrt(2) of its larger number long; sixteen roundings of sines, products and sums
    assert float((m - t).abs().max()) <= (2 ** 0.5 * (2.0 ** -17 + 2.0 ** -18) + 16 * 2.0 ** -24) * float(t.abs().max())


def _observe(lm, cache, seen):
    """Wraps the model's step: counts how many rows of each slot a tracked cache observes."""
    step = lm.model.step

    def counted(c, entries):
        if c is cache:
            most = max(len(e.tokens) for e in entries)
            for e in entries:
                seen[e.slot] = seen.get(e.slot, 0) + (len(e.tokens) if most <= 8 else min(len(e.tokens), 32))
        return step(c, entries)
    lm.model.step = counted


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafted_rows_weigh_once_each(cuda, model_folders, dtype):
    """Drafts that stay: after every step a sequence's scores sum to the rows observed of it, whatever steps brought them."""
    import camelid_b200
    lm = camelid_b200.load(model_folders["tiny_d"], dtype=dtype)
    prompts = [tokens(60 + i, n, 331) for i, n in enumerate([30, 7, 12])]
    cache, seen, looked = lm.new_cache(1024, track_weights=True), {}, []
    _observe(lm, cache, seen)

    def drafter(history):                       # (certain of one token: in float32 it is the model's own, so all drafts stay)
        return known[tuple(history[:1])][len(history):len(history) + 1 + len(history) % 4]
    known = {}
    for p, w in zip(prompts, lm.generate(prompts, max_tokens=24, stop_token_ids=())):
        known[(p[0],)] = list(p) + w
    assert len(known) == 3
    rejected = [0]
    truncate = cache.truncate

    def dropped(slot, length):
        rejected[0] += 1
        return truncate(slot, length)
    cache.truncate = dropped

    def check(live):
        for slot, n in seen.items():
            if not cache.book.slots.is_held(slot):
                continue
            line = torch.cat([cache.scores[0][:, p] for p in cache.book.pages[0][slot]], dim=2)[:, :, :cache.length(slot)].double()
            total = line.sum(2)
            if rejected[0] == 0:
                assert torch.allclose(total, torch.full_like(total, 3.0 * n), rtol=1e-5)
            else:                               # what looked at rejected places went with them, nothing came twice
                assert bool((total <= 3.0 * n * (1 + 1e-5)).all())
            looked.append(slot)
    lm.generate(prompts, max_tokens=24, stop_token_ids=(), drafter=drafter, cache=cache, on_step=check)
    assert len(looked) >= 9 and (dtype == "bfloat16" or rejected[0] == 0)


def test_bfloat16_drafted_tokens_differ_at_near_ties_alone(cuda, model_folders):
    """Where drafted generation first leaves the plain one, the plain run's logits of the two tokens are as near as rounding makes them."""
    import camelid_b200
    lm = camelid_b200.load(model_folders["tiny_d"], dtype="bfloat16")
    prompts = [tokens(80 + i, n, 331) for i, n in enumerate([30, 7, 64, 1])]
    want = lm.generate(prompts, max_tokens=40, stop_token_ids=())
    known = [list(p) + w for p, w in zip(prompts, want)]

    def right(history):
        full = next((k for k in known if k[:len(history)] == history), None)
        return full[len(history):len(history) + 5] if full else []
    got = lm.generate(prompts, max_tokens=40, stop_token_ids=(), drafter=right)
    for p, g, w in zip(prompts, got, want):
        at = next((j for j in range(40) if g[j] != w[j]), None)
        if at is None:
            continue
        cache = lm.new_cache(1024)
        slot = cache.alloc_slot()
        row = lm.step(cache, [camelid_b200.StepEntry(slot, p + w[:at], [len(p) + at - 1])])[0]
        # the caches of one step and of many agree to 4e-2 of the largest logit (as the tracked and the plain cache's do)
        assert float(row[w[at]] - row[g[at]]) <= 2 * 4e-2 * float(row.abs().max())
