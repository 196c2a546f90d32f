"""What stands between two steps, without a device: refusals, the loop with drafted tokens, look-up drafts, the caches that keep
attention weights."""
import random

import pytest
import torch

from camelid_b200 import CacheError, ConfigError, KernelError, PromptLookup, SamplingError, StepError
from camelid_b200.cache import CacheBook, KVSpec, SequenceCache, StateSpec
from camelid_b200.csrc import ops
from camelid_b200.engine.generate import generate
from camelid_b200.engine.model import DecoderModel
from conftest import TINY_A


# ---- the operators' faces -------------------------------------------------------------------------------------------
def test_operators_refuse_cpu_tensors():
    z = lambda *s: torch.zeros(*s)                                          # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)                       # noqa: E731
    with pytest.raises(KernelError):
        ops.attn_paged_weights(z(1, 64), z(1, 64), z(1, 1, 64, 64), z(1, 1, 64, 64), z(1, 1, 64), i(1, 1), i(1), i(1), i(1), 1, 1, 1, 1.0, z(9))
    with pytest.raises(KernelError):
        ops.evict_positions(z(1, 1, 64, 64), None, z(1, 1, 64), i(1, 1), i(1, 1), i(1), i(1), i(1, 1, 4), 0, 0)
    with pytest.raises(KernelError):
        ops.verify_drafts(z(1, 9), i(1), i(1), i(1, 0), None, z(1, 0), z(1), 1.0, 0, 1.0, 0.0, i(1), i(1, 1), i(1), z(64).byte())


def test_scratch_sizes_grow_with_what_they_hold():
    sizes = [ops.attn_weights_floats(n, 8, 2, d, dt, new, length, out) for n in (1, 5) for d in (64, 80) for dt in (torch.bfloat16, torch.float32)
             for new in (1, 9) for length in (1, 700) for out in (False, True)]
    assert min(sizes) > 0
    for dt in (torch.bfloat16, torch.float32):
        assert ops.attn_weights_floats(2, 8, 2, 64, dt, 1, 500, True) <= ops.attn_weights_floats(2, 8, 2, 64, dt, 1, 5000, True)
    assert ops.verify_bytes(0, 0, 100) >= 16 and ops.verify_bytes(4, 2, 5000) >= 4 * (16 * 5 + 8)


def test_scratch_holds_what_one_form_of_the_kernels_keeps():
    """One launch keeps the products, 4 bytes a row and place; several keep the stretches' statistics and outputs and no products."""
    for dtype, rows in ((torch.bfloat16, 4), (torch.bfloat16, 8), (torch.float32, 4), (torch.float32, 8)):
        assert ops.attn_weights_floats(16, 8 * rows, 8, 128, dtype, 1, 32768, True) == 16 * 8 * rows * 32768
        assert ops.attn_weights_floats(3, 8 * rows, 8, 128, dtype, 1, 1000, False) == 3 * 8 * rows * 1024
    for dtype, new in ((torch.float32, 4), (torch.bfloat16, 9)):                # 16 rows in float, 36 on the tensor cores
        few, many = (ops.attn_weights_floats(16, 32, 8, 128, dtype, new, n, False) for n in (2048, 32768))
        assert few <= many < 16 * 32 * new * 2048
    # of 9 to 32 rows on the tensor cores: room for either form (rows of q off 16 bytes take the float kernels)
    split_keys, floats = ops.attn_weights_plan(2, 32, 8, 64, 64, torch.bfloat16, 4, 8192, True)
    splits = -(-8192 // split_keys)
    assert floats == max(2 * 32 * 4 * 8192, 2 * 32 * 4 * (2 + splits * (2 + 64)))


def test_products_are_kept_for_no_more_pages_than_the_cache_has():
    """One long sequence among many short ones does not size the scratch for all."""
    sizes = (64, 32, 8, 128, torch.bfloat16, 8, 131_072, True)
    assert ops.attn_weights_floats(*sizes) == 64 * 8 * 32 * 131_072
    assert ops.attn_weights_floats(*sizes, n_pages=3000) == 8 * 32 * 3000 * 64
    assert ops.attn_weights_floats(*sizes, n_pages=1 << 20) == ops.attn_weights_floats(*sizes)
    assert ops.attn_weights_floats(2, 8, 8, 96, torch.float32, 5, 1000, False, n_pages=20) == 8 * 5 * 20 * 64


def test_kernel_entries_refuse_sizes_before_they_launch():
    """The C entries return the error of a size or type without touching a device."""
    att = ops._fn("attention_weights", "cml_attn_paged_weights")
    good = dict(q=4096, dtype=0, qs=64, out=4096, os=64, k=4096, v=4096, s=4096, so=4096, table=4096, width=1, pages=1, row0=4096, start=4096,
                new=4096, cached=None, n=1, rows=1, heads=1, kv=1, kd=64, vd=64, max_new=1, max_len=1, scale=1.0, split=64, scratch=4096, err=None, stream=None)
    for change, code in (({"dtype": 7}, -2), ({"kd": 24}, -3), ({"kd": 272}, -3), ({"vd": 8}, -3), ({"heads": 3, "kv": 2}, -3), ({"kv": 0}, -3),
                         ({"max_new": 0}, -3), ({"max_len": 0}, -3), ({"split": 0}, -3), ({"split": 63}, -3), ({"scale": 0.0}, -3),
                         ({"scale": float("nan")}, -3), ({"scale": float("inf")}, -3), ({"width": 0}, -3), ({"pages": 0}, -3),
                         ({"n": 70000}, -3), ({"k": 4104}, -4), ({"scratch": 4100}, -4), ({"s": 4104}, -4), ({"n": 0}, 0), ({"rows": 0}, 0)):
        assert att(*{**good, **change}.values()) == code, change
    ev = ops._fn("eviction", "cml_evict_positions")
    good = dict(k=4096, v=4096, s=4096, dtype=0, table=4096, width=1, out=4096, ow=1, lens=4096, keeps=4096, kept=4096, cap=4, entries=1, pages=1,
                n=1, heads=1, kd=64, vd=64, first=0, recent=0, f=None, rot=0, inter=0, stream=None)
    for change, code in (({"dtype": 7}, -2), ({"kd": 24}, -3), ({"kd": 0}, -3), ({"vd": 20}, -3), ({"kd": 1024}, -3), ({"first": -1}, -3),
                         ({"recent": -1}, -3), ({"f": 4096, "rot": 8}, -3), ({"f": 4096, "rot": 80}, -3), ({"f": 4096, "rot": 0}, -3),
                         ({"heads": 0}, -3), ({"width": 0}, -3), ({"ow": 0}, -3), ({"pages": 1 << 30}, -3), ({"k": 4104}, -4), ({"v": 4100}, -4),
                         ({"entries": 1 << 20, "n": 1 << 10}, -3), ({"cap": 0}, 0), ({"n": 0}, 0)):
        assert ev(*{**good, **change}.values()) == code, change
    ve = ops._fn("verify", "cml_verify_drafts")
    good = dict(l=4096, ld=10, rows=1, vocab=10, row0=4096, lens=4096, d=4096, dld=1, p=None, ps=0, pst=0, a=4096, ald=1, nd=4096, n=1, width=1, t=1.0,
                k=0, tp=1.0, mp=0.0, c=4096, tok=4096, err=4096, scratch=4096, stream=None)
    for change, code in (({"vocab": 0}, -3), ({"vocab": (1 << 30) + 1}, -3), ({"t": -1.0}, -3), ({"t": float("nan")}, -3), ({"t": float("inf")}, -3),
                         ({"width": -1}, -3), ({"width": 70000}, -3), ({"rows": -1}, -3), ({"rows": 1 << 30}, -3), ({"n": 1 << 29}, -3),
                         ({"scratch": 4100}, -4), ({"n": 0}, 0)):
        assert ve(*{**good, **change}.values()) == code, change


def test_eviction_refuses_scores_that_do_not_begin_on_eight_bytes():
    ev = ops._fn("eviction", "cml_evict_positions")
    args = [4096, 4096, 4100, 0, 4096, 1, 4096, 1, 4096, 4096, 4096, 4, 1, 1, 1, 1, 64, 64, 0, 0, None, 0, 0, None]
    assert ev(*args) == -4


# ---- caches that keep attention weights --------------------------------------------------------------------------------
def _cache(specs, **kw):
    return SequenceCache(specs, [None] * len(specs), max_tokens=256, max_position=1000, dtype=torch.float32, device="cpu", **kw)


def test_cache_keeps_scores_beside_its_keys():
    spec = KVSpec(2, 32)
    plain, tracked = _cache([spec, spec]), _cache([spec, spec], track_weights=True)
    assert plain.scores is None and plain.scores_of(0) is None
    assert [tuple(t.shape) for t in tracked.scores] == [(2, 4, 2, 64)] and tracked.scores_of(1).shape == (4, 2, 64)
    assert tracked.bytes == plain.bytes + 2 * 4 * 2 * 64 * 4
    for specs in ([KVSpec(2, 32, window=64)], [KVSpec(2, 32, chunk=64)], [spec, StateSpec((3,))], [StateSpec((3,))]):
        with pytest.raises(CacheError):
            _cache(specs, track_weights=True)


def test_only_mixers_that_keep_weights_are_tracked():
    from camelid_b200.parts.attention import GroupedQueryAttention

    class Silent(GroupedQueryAttention):
        def forward(self, ctx, x, residual):
            super().forward(ctx, x, residual)

    class Other(GroupedQueryAttention):
        def tensor_specs(self):
            return super().tensor_specs()

    assert GroupedQueryAttention.keeps_weights and Other.keeps_weights and not Silent.keeps_weights
    model = DecoderModel.from_config(TINY_A, device="cpu")
    assert model.new_cache(128, track_weights=True).scores is not None
    odd = {**TINY_A, "head_dim": 16}
    model = DecoderModel.from_config(odd, device="cpu")
    model.blocks[0].mixer.position.rotary_dim = 8
    with pytest.raises(ConfigError):
        model.new_cache(128, track_weights=True)
    from fomatar_models import CONFIGS as FOMATAR
    with pytest.raises((ConfigError, CacheError)):
        DecoderModel.from_config(FOMATAR["mixed"], device="cpu").new_cache(128, track_weights=True)


def test_a_mixer_with_attention_of_its_own_is_not_tracked():
    """In a tracked cache steps of few tokens run the weighing kernel in place of ``_attend``: a class that changes what that does has to
    say that it keeps weights."""
    from camelid_b200.parts.attention import GroupedQueryAttention

    class Own(GroupedQueryAttention):
        def _attend(self, ctx, q, out, *rest, **kw):
            super()._attend(ctx, q, out, *rest, **kw)

    class Said(Own):
        keeps_weights = True
    assert not Own.keeps_weights and Said.keeps_weights
    model = DecoderModel.from_config(TINY_A, device="cpu")
    model.blocks[0].mixer.__class__ = Own
    with pytest.raises(ConfigError):
        model.new_cache(128, track_weights=True)


def test_evict_refuses_before_anything_changes():
    model = DecoderModel.from_config(TINY_A, device="cpu")
    cache = model.new_cache(128)
    slot = cache.alloc_slot()
    with pytest.raises(CacheError):
        model.evict(cache, [slot], 8)
    cache = model.new_cache(256, track_weights=True)
    slot = cache.alloc_slot()
    cache.book.extend(slot, 100)
    cache.book.commit(slot, 100)
    for args, kw in ((([slot], 0), {}), (([slot], 8), {"first": -1}), (([slot], 8), {"recent": 9}), (([slot], 8), {"first": 5, "recent": 4}),
                     (([slot, slot], 8), {}), (([slot, 3], 8), {})):
        with pytest.raises(CacheError):
            model.evict(cache, *args, **kw)
    assert cache.length(slot) == 100
    assert model.evict(cache, [slot], 100) == [100]                        # nothing to do: no kernel runs
    cache.book.audit()


def test_evict_turns_keys_as_the_mixer_wrote_them(monkeypatch):
    """The dense mixer's kernels pair a channel with the one half the rotary size on, whatever the position encoding calls its pairs; a
    mixer that does not say how it pairs goes by the encoding."""
    model = DecoderModel.from_config(TINY_A, device="cpu")
    for b in model.blocks:
        b.mixer.position.pairing = "interleaved"
        b.mixer.position.load({}, "cpu", torch.float32)
    cache = model.new_cache(256, track_weights=True)
    turned = []
    monkeypatch.setattr(ops, "evict_positions", lambda *args, interleaved, **kw: turned.append(interleaved))

    def once():
        slot = cache.alloc_slot()
        cache.book.extend(slot, 100)
        cache.book.commit(slot, 100)
        assert model.evict(cache, [slot], 8) == [8]
        cache.free_slot(slot)
        now = list(turned)
        turned.clear()
        return now
    assert once() == [False]                                                # all layers turn alike: one call
    model.blocks[0].mixer.key_pairing = ""
    assert sorted(once()) == [False] * (len(model.blocks) - 1) + [True]


# ---- drafted tokens -----------------------------------------------------------------------------------------------------
class Rolling:
    """A cache of the bookkeeping alone."""
    state = []

    def __init__(self, n_pages=16, n_slots=8):
        self.book = CacheBook([KVSpec(1, 16)], n_pages, n_slots, 10_000)

    def alloc_slot(self):
        return self.book.alloc_slot()

    def free_slot(self, s):
        self.book.free_slot(s)

    def length(self, s):
        return self.book.length[s]

    def truncate(self, s, n):
        self.book.truncate(s, n)


class Counting:
    """The next token is (7 * last + position) % 50; keeps what each slot holds, as a cache would."""

    def __init__(self):
        self.held, self.steps, self.layouts = {}, 0, set()

    def step(self, cache, entries):
        self.steps += 1
        self.layouts.add(tuple(len(e.tokens) for e in entries))
        cache.book.check_extend([(e.slot, len(e.tokens)) for e in entries])
        rows = []
        for e in entries:
            start = cache.book.length[e.slot]
            held = self.held.setdefault(e.slot, [])[:start] if start else []
            assert len(held) == start
            cache.book.extend(e.slot, len(e.tokens))
            cache.book.commit(e.slot, len(e.tokens))
            self.held[e.slot] = held + list(e.tokens)
            rows += [(7 * self.held[e.slot][start + w] + start + w) % 50 for w in e.want]
        return rows


class Exact:
    """Verifies greedily."""
    vocab_size = 50

    def sample(self, logits, histories):
        return list(logits)

    def verify(self, logits, drafts, histories, probs=None, row0=None):
        counts, nexts = [], []
        for d, at in zip(drafts, row0):
            rows = logits[at:at + len(d) + 1]
            n = 0
            while n < len(d) and d[n] == rows[n]:
                n += 1
            counts.append(n)
            nexts.append(rows[n])
        return counts, nexts


def _expected(history):
    out, h = [], list(history)
    for _ in range(6):
        h.append((7 * h[-1] + len(h) - 1) % 50)
        out.append(h[-1])
    return out


@pytest.mark.parametrize("stops", [set(), {4, 13}])
def test_drafted_loop_gives_the_plain_loops_tokens(stops):
    rng = random.Random(0)
    prompts = [[1, 2, 3], [40], [7] * 70, [9, 8]]
    want = [r.tokens for r in generate(Counting(), Rolling(), Exact(), prompts, 40, stop_ids=stops)]
    reasons = [r.finish_reason for r in generate(Counting(), Rolling(), Exact(), prompts, 40, stop_ids=stops)]

    def partly(history):
        d = _expected(history)
        if rng.random() < 0.6:
            d[rng.randrange(len(d))] += 1
        return [t % 50 for t in d[:rng.randrange(7)]]
    steps = {}
    for name, drafter in (("right", _expected), ("none", lambda h: []), ("wrong", lambda h: [(t + 1) % 50 for t in _expected(h)]), ("partly", partly),
                          ("lookup", PromptLookup(4, 2)), ("tensor", lambda h: (torch.tensor(_expected(h)), None))):
        model, cache = Counting(), Rolling()
        got = generate(model, cache, Exact(), prompts, 40, stop_ids=stops, drafter=drafter, max_batch=3)
        assert [r.tokens for r in got] == want, name
        assert [r.finish_reason for r in got] == reasons, name
        cache.book.audit()
        assert cache.book.slots.n_held == 0
        steps[name] = model.steps
        if name == "right" and not stops:
            assert len(model.layouts) <= 14         # what a captured step is kept by: not one for every mix of drafts
    if not stops:
        assert steps["right"] < steps["none"] / 4 and steps["wrong"] == steps["none"]


def test_drafted_loop_keeps_within_budget_and_cache():
    model, cache = Counting(), Rolling(n_pages=2)
    out = generate(model, cache, Exact(), [[1] * 120], 50, drafter=_expected)
    assert len(out[0].tokens) == 9 and out[0].finish_reason == "capacity"
    assert [r.tokens for r in generate(Counting(), Rolling(n_pages=2), Exact(), [[1] * 120], 50)] == [out[0].tokens]
    assert generate(Counting(), Rolling(), Exact(), [[1]], 0, drafter=_expected)[0].tokens == []


def test_drafted_loop_brings_no_rows_of_its_own_where_weights_are_kept():
    """Rows that only make steps of one size would leave their weights in the scores."""
    model, cache = Counting(), Rolling()
    cache.scores = [torch.zeros(1)]
    drafts = {1: [5, 6, 7], 2: [], 3: [9]}
    generate(model, cache, Exact(), [[1], [2], [3]], 6, drafter=lambda h: drafts[h[0]])
    assert (4, 1, 2) in model.layouts and (4, 4, 4) not in model.layouts


def test_drafted_loop_refusals():
    with pytest.raises(StepError):
        generate(Counting(), Rolling(), Exact(), [[1]], 5, drafter=lambda h: [50])
    cache = Rolling()
    cache.state = [torch.zeros(1)]
    with pytest.raises(StepError):
        generate(Counting(), cache, Exact(), [[1]], 5, drafter=_expected)
    cache = Rolling()
    cache.book.kv_specs = [KVSpec(1, 16, window=64)]
    with pytest.raises(StepError):
        generate(Counting(), cache, Exact(), [[1]], 5, drafter=_expected)
    cache = Rolling()
    with pytest.raises(ValueError):
        generate(Counting(), cache, Exact(), [[1]], 5, drafter=lambda h: ["x"])
    assert cache.book.slots.n_held == 0


def test_verification_refuses_rows_that_two_sequences_adjust():
    """A row is adjusted in place by one history: two sequences that name it would get one answer for both."""
    from camelid_b200.sampling import Sampler, SamplingOptions
    sampler = Sampler(SamplingOptions(temperature=0.5, repeat_penalty=1.2, seed=1), 10, "cpu")
    logits = torch.zeros(3, 10)
    for drafts, row0 in (([[1], [2]], [0, 1]), ([[1], []], [0, 0]), ([[], []], [2, 2])):
        with pytest.raises(SamplingError):
            sampler.verify(logits, drafts, [[3], [4]], row0=row0)
    assert bool((logits == 0).all())


def test_certain_drafts_outside_the_vocabulary_beside_probabilities(monkeypatch):
    """A draft that is no token reaches the kernel, which rejects and reports it, whatever the other sequences bring."""
    from camelid_b200.sampling import Sampler, SamplingOptions
    sampler = Sampler(SamplingOptions(temperature=0.5, seed=1), 10, "cpu")
    given = []

    def verify(logits, row0, lens, drafts, probs, accept, draws, *rest):
        given.append((drafts.tolist(), probs))
        counts, tokens = rest[4], rest[5]
        counts.zero_(), tokens.zero_()
    monkeypatch.setattr(ops, "verify_drafts", verify)
    certain = [[10, 3], [-1, 2]]
    for d in certain:
        sampler.verify(torch.zeros(5, 10), [[4], d], [[1], [2]], [torch.full((1, 10), 0.1), None])
        drafts, probs = given.pop()
        want = torch.zeros(2, 10)
        want[1, d[1]] = 1.0
        assert drafts == [[4, 0], d] and torch.equal(probs[1], want) and bool((probs[0, 0] == 0.1).all())


def test_lookup_drafts():
    look = PromptLookup(3, 2)
    assert look([]) == [] and look([5]) == [] and look([1, 2, 3]) == []
    assert look([5, 5]) == [5] and look([1, 2, 9, 1, 2]) == [9, 1, 2]
    assert look([1, 2, 7, 8, 1, 2, 9, 8, 1, 2]) == [9, 8, 1]               # the last occurrence
    assert look([4, 2, 7, 3, 2]) == [7, 3, 2]                               # no pair, but the single token
    rng = random.Random(1)
    for _ in range(200):
        h = [rng.randrange(4) for _ in range(rng.randrange(12))]
        want = []
        for size in range(min(2, len(h) - 1), 0, -1):
            places = [a for a in range(len(h) - size) if h[a:a + size] == h[-size:]]
            if places:
                want = h[places[-1] + size:][:3]
                break
        assert look(h) == want, h
    for bad in ((0, 1), (1, 0)):
        with pytest.raises(SamplingError):
            PromptLookup(*bad)
