"""The memory plan: bytes of weights, cache and workspace from a configuration alone, and the
refusal before anything is allocated."""
import pytest
import torch

import camelid_b200
from camelid_b200 import MemoryBudgetError, benchmark, memory_plan
from conftest import TINY_A, TINY_B


def test_plan_counts_what_the_survey_counts():
    """Llama 3.2 1B: 973.1 M linear + 262.7 M embedding (tied) + 67.6 k norm parameters; the
    cache keeps 2 * 16 layers * 8 kv heads * 64 = 16,384 elements a position."""
    cfg = benchmark.config_for(2)
    p = memory_plan(cfg, "bfloat16", max_tokens=8 * 4096, max_slots=8)
    assert p.weights == (973_078_528 + 262_668_288 + 33 * 2048) * 2
    assert p.cache == 8 * 4096 * 16_384 * 2
    assert p.total == p.weights + p.cache + p.workspace and 0 < p.workspace < 1 << 30
    f = memory_plan(cfg, "float32", max_tokens=8 * 4096, max_slots=8)
    assert f.weights == 2 * p.weights and f.cache == 2 * p.cache
    untied = memory_plan({**cfg, "tie_word_embeddings": False}, "bfloat16")
    assert untied.weights - p.weights == 262_668_288 * 2 and untied.cache == 0
    # tokens are rounded up to pages of 64
    assert memory_plan(TINY_A, "float32", max_tokens=65).cache == memory_plan(TINY_A, "float32", max_tokens=128).cache


def test_8b_in_float32_is_refused_on_a_32_gb_device_with_the_numbers():
    cfg = benchmark.config_for(4)
    plan = memory_plan(cfg, "float32", max_tokens=8 * 8192, max_slots=8)
    assert 32.0e9 < plan.weights < 32.3e9                      # 8.03 G parameters in 4 bytes
    with pytest.raises(MemoryBudgetError) as e:
        plan.check(32 * 2 ** 30, "Llama 3.1 8B in float32")
    assert e.value.needed == plan.total and e.value.available == 32 * 2 ** 30
    assert f"{plan.weights:,}" in str(e.value) and f"{plan.cache:,}" in str(e.value)
    plan.check(64 * 2 ** 30)
    assert isinstance(e.value, camelid_b200.CacheError) and isinstance(e.value, camelid_b200.CamelidError)


def test_load_refuses_before_it_reads_a_tensor():
    """``load_tensors`` checks names, shapes and then the bytes: a source whose tensors would
    not fit is refused without one tensor having been asked for."""
    from camelid_b200 import DecoderModel
    model = DecoderModel.from_config(TINY_B, dtype=torch.float32, device="cpu")
    specs = model.tensor_specs()

    class Source:
        asked = []

        def names(self):
            return list(specs)

        def shape(self, name):
            return list(specs[name].shape)

        def dtype(self, name):
            return torch.bfloat16

        def tensor(self, name):
            self.asked.append(name)
            raise AssertionError("no tensor may be read")
    src = Source()
    need = model.memory_plan().weights
    with pytest.raises(MemoryBudgetError) as e:
        model.load_tensors(src, available_bytes=need - 1)
    assert src.asked == [] and not model.loaded and e.value.needed == need


def test_chunked_portions_and_their_scratch():
    """Tiles of the portions that run by chunks and of no other; the bound on their number holds for every mix; the plan
    counts what single tokens and ragged portions beside a prompt take."""
    import random
    from camelid_b200.config.plan import PartSpec
    from camelid_b200.csrc import ops
    from camelid_b200.engine.context import StepContext
    from camelid_b200.parts import build_part
    rng = random.Random(5)
    for _ in range(300):
        news = [int(2 ** rng.uniform(0, 9)) for _ in range(rng.randint(1, 40))]
        if max(news) == 1:
            continue
        size, least = key = rng.choice(((64, 128), (64, 64), (64, 32), (32, 128)))
        layout, host, _, _ = StepContext.host_arrays(range(len(news)), [0] * len(news), [[0] * n for n in news], [[] for _ in news], [], [64, key])
        for r, floor in ((64, 1), (key, least)):
            want = [(s, q) for s, n in enumerate(news) for q in range(0, n, r if floor == 1 else size) if n >= floor]
            assert list(zip(layout.view(host, f"tile_seq{r}"), layout.view(host, f"tile_q0{r}"))) == want and layout.n_tiles[r] == len(want)
        assert len(want) <= ops.chunks_at_most(sum(news), len(news), size, least)
    common = {"hidden_size": 64, "num_heads": 16, "key_dim": 128, "value_dim": 128, "state_size": 128, "conv_taps": 4, "gate_cap": 15.0}
    square = 64 * 64
    floats = {"retention": 16 * (square + 4 * 64 + 128 * 128), "matrix_memory": 16 * (square + 4 * 64 + 129 * 128),
              "state_space": square + 16 * (3 * 64 + 128 * 128), "gated_delta": 16 * ops.gated_chunk_floats(128, 128)}
    for kind, per_chunk in floats.items():
        part = build_part("mixer", PartSpec(kind, {**common, "decay": [0.9] * 16 if kind == "retention" else None}))
        size, least = part.query_tile_sizes()[0]
        for news in ([128] + [1] * 63, [2048] + [1] * 200, [least] * 40, [least + 1] * 30, [2047]):
            assert part.workspace(sum(news), len(news)) >= 4 * per_chunk * sum(-(-n // size) for n in news if n >= least)


def test_shares_of_single_tokens_over_a_latent():
    """Every multiprocessor gets at most two blocks, a row at most 64 shares; the plan counts what the shares take."""
    import random
    from camelid_b200.config.plan import PartSpec
    from camelid_b200.csrc import ops
    from camelid_b200.parts import build_part
    from camelid_b200.parts.latent_attention import pages_a_block
    rng = random.Random(6)
    for _ in range(500):
        pages, rows, heads = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 9)), rng.choice((1, 16, 64, 65, 128))
        part = build_part("mixer", PartSpec("latent_attention", {"hidden_size": 64, "num_heads": heads, "head_dim": 32, "value_dim": 32, "rank": 96, "rot_dim": 0}))
        windowed = rng.random() < 0.5
        per = pages_a_block(pages, rows * part.row_blocks, ops.SMS, windowed)
        assert 0 <= per < max(pages, 1)
        if per:
            shares = -(-pages // per)
            assert 1 < shares <= 64 and rows * part.row_blocks * shares <= 2 * ops.SMS
            assert part.workspace(rows, rows) >= 4 * shares * rows * heads * (96 + 2)
        else:
            assert pages < 4 or rows * part.row_blocks * 2 > ops.SMS
    assert pages_a_block(32, 1, 148) == 1 and pages_a_block(128, 1, 148) == 2 and pages_a_block(8, 128, 148) == 0
    assert [pages_a_block(p, 2, 148, True) for p in (4, 9, 17)] == [2, 3, 3] and pages_a_block(9, 128, 148, True) == 6


def test_plan_counts_scores_and_scratch_of_a_cache_that_keeps_weights():
    from camelid_b200 import DecoderModel
    cfg = benchmark.config_for(2)                              # 16 layers, 8 kv heads of 64, 4 heads each
    sizes = dict(max_tokens=8 * 4096, max_slots=8)
    plain, tracked = memory_plan(cfg, "bfloat16", **sizes), memory_plan(cfg, "bfloat16", **sizes, track_weights=True)
    scores = 4 * 16 * 8 * 8 * 4096
    assert tracked.cache == plain.cache + scores and tracked.weights == plain.weights
    # the products of 8 new tokens of 4 heads for every cached position, and the scores once more beside a capture
    assert tracked.workspace >= plain.workspace + scores + 4 * 8 * 32 * 8 * 4096
    assert tracked.workspace < plain.workspace + scores + 4 * 8 * 32 * 8 * 4096 + (32 << 20)
    model = DecoderModel.from_config(TINY_B, dtype=torch.float32, device="cpu")
    plan, bare = (model.memory_plan(1024, 4, track_weights=t) for t in (True, False))
    cache, without = (model.new_cache(1024, 4, track_weights=t) for t in (True, False))
    assert cache.bytes - without.bytes == 4 * sum(t.numel() for t in cache.scores) + 4 * cache.weights_scratch.numel()
    assert plan.total - bare.total == cache.bytes - without.bytes + 4 * sum(t.numel() for t in cache.scores)
    assert without.weights_scratch is None and cache.weights_scratch.numel() == model.weights_scratch(16, 4)


def test_new_cache_refuses_scores_and_scratch_that_do_not_fit(monkeypatch):
    from camelid_b200 import DecoderModel, memory
    model = DecoderModel.from_config(TINY_B, dtype=torch.float32, device="cpu")
    need = {t: (lambda p: p.cache + p.workspace)(model.memory_plan(4096, 8, track_weights=t)) for t in (True, False)}
    monkeypatch.setattr(memory, "device_free_bytes", lambda device: need[True] - 1)
    model.new_cache(4096, 8)
    with pytest.raises(MemoryBudgetError) as e:
        model.new_cache(4096, 8, track_weights=True)
    assert e.value.needed == need[True] > need[False]
    monkeypatch.setattr(memory, "device_free_bytes", lambda device: need[True])
    model.new_cache(4096, 8, track_weights=True)


def test_one_scratch_serves_every_step_of_a_cache():
    """The bound holds for any number of sequences, new tokens, heads and table widths; it follows the cache's pages."""
    import random
    from camelid_b200.csrc import ops
    rng = random.Random(3)
    for _ in range(4000):
        kv, group = rng.choice((1, 2, 3, 5, 8, 16, 40)), rng.choice((1, 2, 3, 4, 6, 8, 16))
        dim, dtype = rng.choice((16, 64, 96, 128, 256)), rng.choice((torch.bfloat16, torch.float32))
        slots, n_pages = int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(0, 13))
        most, with_output = rng.choice(((8, True), (32, False)))
        room = ops.attn_weights_room(slots, n_pages, kv * group, kv, dim, dtype, most, with_output)
        for _ in range(10):
            n, new, width = rng.randint(1, slots), rng.randint(1, most), int(2 ** rng.uniform(0, 14))
            floats = ops.attn_weights_plan(n, kv * group, kv, dim, dim, dtype, new, width * 64, with_output, n_pages, True)[1]
            assert floats <= room, (kv, group, dim, dtype, slots, n_pages, n, new, width, with_output)
    assert ops.attn_weights_room(64, 4096, 32, 8, 128, torch.bfloat16, 8, True) == 8 * 32 * 4096 * 64


def test_memory_command_of_a_tracked_cache(tmp_path, capsys):
    import json
    from camelid_b200 import cli
    path = tmp_path / "config.json"
    path.write_text(json.dumps(TINY_B))
    plans = []
    for more in ([], ["--track-weights"]):
        assert cli.main(["memory", str(path), "--dtype", "float32", "--max-tokens", "1024", "--max-slots", "4", *more]) == 0
        plans.append(json.loads(capsys.readouterr().out))
    want = memory_plan(TINY_B, "float32", max_tokens=1024, max_slots=4, track_weights=True).as_dict()
    assert {k: plans[1][k] for k in want} == want and plans[1]["cache"] > plans[0]["cache"]
