"""The engine over a cache held in 8 bits: however the work is cut, against the plain implementation whose keys and values
are rounded to the same codes; forks, captured steps, generation, the command line, and what is refused."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_mekazen
import plain_qwen3 as plain
import replay_helpers as cuts
from conftest import ROOT, TOL_BF16_VS_EXACT, random_ids

gpu = pytest.mark.gpu
LIMITS = {"fp8": 448.0, "int8": 127.0}
LENGTHS = {"A": [5, 31, 100], "B": [1, 40, 130], "C": [3, 200, 33], "D": [300, 2, 257]}
# float32: the plain side holds the same codes but where a quotient lies within the engine's 32-bit error of the middle
# between two. Such a code moves one number of one key or value by one step, a sixteenth of the row's largest at most, and
# a logit of these models (below 2 in magnitude) by a small part of that: far less than this.
TOL_CODES_F32 = 1e-2


def coded(rows, codes):
    """float64 rows as a cache in 8 bits holds them."""
    scale = (np.abs(rows).max(-1, keepdims=True).astype(np.float32) / np.float32(LIMITS[codes])).astype(np.float64)
    y = rows / np.where(scale > 0, scale, 1.0)
    if codes == "int8":
        return np.clip(np.round(y), -127, 127) * scale
    step = np.ldexp(1.0, np.maximum(np.frexp(y)[1], -5) - 4)
    return np.clip(np.round(y / step) * step, -448, 448) * scale


@pytest.fixture(scope="module")
def references(model_folders):
    """(model, codes) -> (requests, logits with coded keys and values, largest change the codes make)."""
    made, original = {}, plain.causal_gqa_attention

    def of(name, codes):
        if (name, codes) not in made:
            _, config, tensors, _ = model_folders[name]
            requests = {f"r{i}": random_ids(100 * i + len(name), n, config["vocab_size"]) for i, n in enumerate(LENGTHS[name])}
            bare = {k: plain.forward_logits(config, tensors, ids) for k, ids in requests.items()}
            plain.causal_gqa_attention = lambda q, k, v, scale, window=None: original(q, coded(k, codes), coded(v, codes), scale, window)
            try:
                exact = {k: plain.forward_logits(config, tensors, ids) for k, ids in requests.items()}
            finally:
                plain.causal_gqa_attention = original
            shift = max(float(np.abs(exact[k] - bare[k]).max()) for k in requests)
            made[(name, codes)] = (requests, exact, shift)
        return made[(name, codes)]
    return of


def make_engine(model_folders, name, dtype, codes, pages=256, **options):
    from metallix_b200.engine import Engine
    folder, _, _, page = model_folders[name]
    return Engine.from_folder(folder, dtype=dtype, page_tokens=page, num_pages=pages, max_requests=8, cache_dtype=codes, **options)


def limit_of(dtype, shift):
    # bfloat16: rows that differ by 2^-8 get other codes here and there, each off by what the codes are off anyway
    return TOL_CODES_F32 if dtype == "float32" else TOL_BF16_VS_EXACT + 2 * shift


# ----------------------------------------------------------------- without a GPU
def test_bytes_of_pages_of_codes():
    from metallix_b200.cache import PagedCache
    from metallix_b200.config.spec import CacheNeed
    full = CacheNeed(kind="kv_pages", kv_heads=2, head_dim=64, codes="fp8")
    window = CacheNeed(kind="kv_pages", kv_heads=2, head_dim=64, window=8, codes="fp8")
    bare = CacheNeed(kind="kv_pages", kv_heads=2, head_dim=64)
    rows = 2 * 2 * 16     # of a page: planes, heads, positions
    # codes and scales of every entry, and one buffer for pages read back per shape
    assert PagedCache.page_bytes([full, full, window], 16, torch.bfloat16) == rows * (3 * (64 + 4) + 64 * 2)
    assert PagedCache.page_bytes([bare, bare], 16, torch.bfloat16) == rows * 2 * 64 * 2
    assert full.group_key() != bare.group_key()
    cache = PagedCache([full, window, bare], 16, 4, 2, torch.bfloat16, "cpu", allocate=False)
    assert cache.bytes_per_token() == 2 * 2 * (2 * (64 + 4) + 64 * 2)


def test_the_attention_lists_what_is_read_back():
    from metallix_b200.parts import StepPlan
    from metallix_b200.parts.attention import attention_tiles
    made = attention_tiles(StepPlan([5, 1, 300, 1], [0, 7, 2000, 0], 4, 2300)).arrays
    assert [made[f"read_{name}"].tolist() for name in ("request", "first", "last")] == [[0, 2], [0, 2000], [4, 2299]]
    graph = attention_tiles(StepPlan([1, 1, 1, 1], None, 2, 4096, replayable=True)).arrays
    assert all(graph[f"read_{name}"].size == 0 for name in ("request", "first", "last"))


def test_single_tokens_over_codes_need_their_kernel():
    """A mixer that asks for the general kernel over codes is told so, ahead of any launch."""
    from metallix_b200 import ops
    from metallix_b200.config.spec import CacheNeed
    from metallix_b200.parts.attention import attend_cached
    from metallix_b200.parts.registry import CacheView

    pool = object.__new__(ops.QuantizedPool)     # as if on a device
    pool.shape = torch.Size((3, 2, 1, 4, 8))

    class Context:
        extras = {"attention_tiles": {"multi_tiles": 0, "decode_rows": 1, "read_request": torch.zeros(0)}}
    view = CacheView(need=CacheNeed("kv_pages"), pool=pool)
    with pytest.raises(ValueError, match="split-key"):
        attend_cached(torch.zeros(1, 2, 8), view, Context(), scale=1.0)


# ----------------------------------------------------------------- the engine
@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_every_cut_matches_the_plain_implementation(model_folders, references, name, dtype, codes):
    from metallix_b200.engine import StepEntry
    requests, exact, shift = references(name, codes)
    limit = limit_of(dtype, shift)
    engine = make_engine(model_folders, name, dtype, codes)
    whole_steps = cuts.whole(requests)
    for label, steps in (("whole", whole_steps), ("tail", cuts.tail_by_one(requests)), ("ragged", cuts.ragged(requests)),
                         ("whole, captured", whole_steps + whole_steps), ("ragged, captured", cuts.ragged(requests))):
        worst, _ = cuts.replay(engine, steps, exact, StepEntry)
        assert worst < limit, f"{label}: {worst}"
    engine.manager.check_invariants()
    held = engine.cache.groups[0]
    assert held.pool.dtype == {"fp8": torch.float8_e4m3fn, "int8": torch.int8}[codes] and held.scales.isfinite().all()


@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "D"])
def test_mixed_batches_with_pages_used_again(model_folders, references, name, dtype, codes):
    from metallix_b200.engine import StepEntry
    requests, exact, shift = references(name, codes)
    page = model_folders[name][3]
    for seed in (0, 1):
        steps, peak = cuts.mixed(requests, seed)
        engine = make_engine(model_folders, name, dtype, codes, pages=peak // page)
        worst, _ = cuts.replay(engine, steps, exact, StepEntry)
        assert worst < limit_of(dtype, shift), f"seed {seed}: {worst}"


@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
def test_the_first_layers_rows_are_the_nearest_codes(model_folders, codes):
    """What a bfloat16 engine without codes holds of the first layer, and what one with codes holds: values code for code,
    keys but for the rounding that the first one's pages have and the second's codes have not."""
    from metallix_b200.engine import StepEntry
    ids = random_ids(5, 61, model_folders["D"][1]["vocab_size"])
    engines = [make_engine(model_folders, "D", "bfloat16", kind) for kind in (None, codes)]
    for engine in engines:
        engine.step([StepEntry("r", ids[:60], [59])])
        engine.step([StepEntry("r", ids[60:], [0])])
        engine.check()
    bare, held = (engine.cache.groups[0] for engine in engines)
    table = engines[0].manager.table(engines[0]._ids["r"], 0)
    assert table == engines[1].manager.table(engines[1]._ids["r"], 0)
    page = bare.page_tokens
    for position in range(61):
        at = (0, table[position // page], slice(None), slice(None), position % page)
        rows = bare.pool[at].double()
        scale, code = held.scales[at].double(), held.pool[at].float().double()
        largest = rows.abs().amax(-1)
        expect = torch.from_numpy(coded(rows.cpu().numpy(), codes)).cuda()
        assert torch.equal((code * scale.unsqueeze(-1))[1], expect[1])
        assert ((scale[0] * LIMITS[codes] - largest[0]).abs() <= 2.0 ** -7 * largest[0]).all()
        half = (largest / 254 if codes == "int8" else largest / 28).unsqueeze(-1)      # of the widest step
        assert ((code[0] * scale[0].unsqueeze(-1) - rows[0]).abs() <= half[0] + 2.0 ** -7 * largest[0].unsqueeze(-1)).all()


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forks_share_codes_and_scales(model_folders, references, dtype):
    from metallix_b200.engine import StepEntry
    requests, exact, shift = references("D", "fp8")
    ids, limit = requests["r2"], limit_of(dtype, shift)
    engine = make_engine(model_folders, "D", dtype, "fp8")
    engine.step([StepEntry("parent", ids[:37], [36])])     # ends inside a page
    engine.fork("parent", "child")
    other = random_ids(9, 20, model_folders["D"][1]["vocab_size"])
    for at in range(20):                                   # the parent goes its own way first
        engine.step([StepEntry("parent", [other[at]], [0])])
    engine.release("parent")
    for at in range(37, 80):
        logits = engine.step([StepEntry("child", [ids[at]], [0])])
        assert np.abs(logits.cpu().double().numpy()[0] - exact["r2"][at]).max() < limit
    engine.check()


@gpu
def test_generation_over_codes(model_folders):
    """Through the scheduler with too few pages for all: the same tokens as with enough."""
    from metallix_b200.engine.generate import generate
    prompts = [random_ids(i, 20 + 7 * i, model_folders["D"][1]["vocab_size"]) for i in range(4)]
    picked = [[r.generated_ids for r in generate(make_engine(model_folders, "D", "float32", "int8", pages=pages), prompts,
                                                 max_new_tokens=24, ignore_eos=True)] for pages in (64, 12)]
    assert picked[0] == picked[1] and all(len(ids) == 24 for ids in picked[0])


@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
@pytest.mark.parametrize("name,dtype", [("small", "float32"), ("wide", "float32"), ("wide", "bfloat16")])
def test_chunks_gates_and_projection_norms_over_codes(tmp_path, name, dtype, codes):
    """Another decoder design: the norm over the whole projection, neighbouring pairs turned, values from the raw keys,
    chunks, a gate. Its logits move by no more than 8-bit rows move them, and cuts agree among one another."""
    import test_mekazen
    from metallix_b200.engine import Engine, StepEntry
    raw, seed, page, sharpen = test_mekazen.MODELS[name]
    folder = test_mekazen.write_folder(str(tmp_path / name), raw, seed, sharpen)
    config, tensors = plain_mekazen.read_model(folder)
    requests = {"a": random_ids(3, 75, raw["vocab"]), "b": random_ids(4, 130, raw["vocab"])}
    exact = {k: plain_mekazen.forward_logits(config, tensors, ids) for k, ids in requests.items()}
    engine = Engine.from_folder(folder, dtype=dtype, page_tokens=page, num_pages=96, max_requests=4, cache_dtype=codes)
    # a row's error is at most 2^-4 of a value's magnitude (fp8) or 2^-8 of the row's largest (int8); a few layers of
    # it, against logits of the capped size below, stay within a tenth of their largest
    limit = 0.1 * max(np.abs(e).max() for e in exact.values())
    seen = []
    for steps in (cuts.whole(requests), cuts.tail_by_one(requests), cuts.ragged(requests)):
        worst, logits = cuts.replay(engine, steps, exact, StepEntry)
        assert worst < limit, worst
        seen.append(logits)
    drift = max(float(np.abs(row - seen[0][key]).max()) for other in seen[1:] for key, row in other.items())
    assert drift < (TOL_CODES_F32 if dtype == "float32" else limit), drift


@gpu
def test_the_pool_by_bytes_holds_more_pages(model_folders):
    from metallix_b200.engine import Engine
    folder = model_folders["D"][0]
    pages = [Engine.from_folder(folder, page_tokens=16, pool_bytes=2 ** 24, cache_dtype=codes).cache.groups[0].num_pages
             for codes in (None, "fp8")]
    # 2 layers: 2 x 64 x 2 bytes a row without codes; 2 x 68 and a shared 64 x 2 with them
    assert pages[0] == 2 ** 24 // (2 * 2 * 16 * 256) and pages[1] == 2 ** 24 // (2 * 2 * 16 * (136 + 128))


@gpu
def test_what_is_refused(model_folders, tmp_path):
    from metallix_b200.engine import Engine
    with pytest.raises(ValueError, match="cache_dtype must be"):
        make_engine(model_folders, "A", "bfloat16", "int4")
    import test_zitezen
    from metallix_b200.config import parse_config
    raw = next(iter(test_zitezen.MODELS.values()))[0]
    with pytest.raises(ValueError, match="compute type only"):      # its latent attention caches rows of its own
        Engine.from_random(parse_config(raw), 0, dtype="bfloat16", num_pages=8, cache_dtype="fp8")


@gpu
def test_the_command_line(model_folders):
    folder, config, _, _ = model_folders["D"]
    command = [sys.executable, os.path.join(ROOT, "bin", "mxb"), "gen", "--model", folder, "--input-ids",
               ",".join(map(str, random_ids(1, 40, config["vocab_size"]))), "--max-tokens", "8", "--dtype", "float32", "--ignore-eos",
               "--cache-dtype", "int8"]
    run = subprocess.run(command, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0, run.stderr
    report = json.loads(run.stdout.strip().splitlines()[-1])
    assert len(report["generated_ids"]) == 8
    assert report["logical_kv_bytes"] == report["cached_tokens"] * 2 * 2 * 2 * (64 + 4)      # layers, planes, heads, a row


DESIGNS = [("sadosun", "wide", None), ("sadosun", "bare", None), ("kokolorn", "wide", None), ("kokolorn", "bare", None),
           ("dimorax", "wide", (0, 1, 3)), ("mekuvik", "wide", (0, 3))]


@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design,name,kept", DESIGNS, ids=lambda v: v if isinstance(v, str) else "")
def test_other_designs_attend_to_codes_alike_however_cut(design, name, kept, dtype, codes):
    """Sinks, values turned by position, biases by distance, another layer's keys and values, kept positions, small pages:
    single tokens read the codes, portions read pages back, and both see the same rows."""
    import importlib
    from metallix_b200.config import parse_config
    from metallix_b200.engine import Engine, StepEntry
    raw, seed, page, _ = importlib.import_module(f"test_{design}").MODELS[name]
    if kept is not None:      # without the layers of latent attention, whose rows stay in the compute type
        raw = {**raw, "layers": [raw["layers"][i] for i in kept]}
        if raw.get("loop"):
            raw["loop"] = {**raw["loop"], "start": 0, "stop": len(kept)}
    requests = {"a": random_ids(3, 75, raw["vocab"]), "b": random_ids(4, 190, raw["vocab"])}

    def logits_of(cache_dtype, steps):
        engine = Engine.from_random(parse_config(raw), seed, dtype=dtype, page_tokens=page, num_pages=128, max_requests=4,
                                    cache_dtype=cache_dtype)
        blank = {k: np.zeros((len(ids), raw["vocab"])) for k, ids in requests.items()}
        return cuts.replay(engine, steps, blank, StepEntry)[1]
    plain_rows = logits_of(None, cuts.whole(requests))
    top = max(np.abs(row).max() for row in plain_rows.values())
    seen = [logits_of(codes, steps) for steps in (cuts.whole(requests), cuts.tail_by_one(requests, 40), cuts.ragged(requests))]
    drift = max(float(np.abs(row - seen[0][key]).max()) for other in seen[1:] for key, row in other.items())
    shift = max(float(np.abs(row - plain_rows[key]).max()) for key, row in seen[0].items())
    assert shift > 0.0       # the codes were used
    # float32: as TOL_CODES_F32 says; bfloat16: codes that flip move a logit no further than the codes themselves move it
    assert drift < (TOL_CODES_F32 * max(top, 1.0) if dtype == "float32" else TOL_BF16_VS_EXACT * max(top, 1.0) + 2 * shift), (drift, shift, top)


# Matrices large enough for the float32 products on the tensor cores, so that a second engine's are not the same to the bit.
CHECKED = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", hidden_act="silu", num_hidden_layers=4, hidden_size=1024,
               num_attention_heads=16, num_key_value_heads=8, head_dim=128, intermediate_size=2048, vocab_size=2000,
               rope_theta=10000.0, rms_norm_eps=1e-6, tie_word_embeddings=True, max_position_embeddings=4096)


@gpu
@pytest.mark.parametrize("codes", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_command_line_checks_a_cache_of_codes(tmp_path, dtype, codes):
    """Two engines whose products differ in the last bits code a number here and there otherwise: that is no fault, and
    what the codes themselves move is in the report."""
    path = tmp_path / "config.json"
    path.write_text(json.dumps(CHECKED))
    command = [sys.executable, os.path.join(ROOT, "bin", "mxb"), "gen", "--config", str(path), "--random-weights", "3", "--input-ids",
               ",".join(map(str, random_ids(9, 60, CHECKED["vocab_size"]))), "--max-tokens", "24", "--dtype", dtype, "--ignore-eos",
               "--num-pages", "64", "--cache-dtype", codes, "--verify-cache"]
    run = subprocess.run(command, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=600, cwd=ROOT)
    assert run.returncode == 0, (run.stdout[-2000:], run.stderr[-2000:])
    report = json.loads(run.stdout.strip().splitlines()[-1])["cache_comparisons"]
    assert report["logits_within_bound"] is True and report["positions"] == 24
    assert 0.0 < report["max_abs_logit_shift_of_codes"] and report["max_abs_logit_difference"] <= 2 * report["max_abs_logit_shift_of_codes"] + (
        5e-4 if dtype == "float32" else 2.5e-2 * report["max_abs_logit_difference"] / report["max_difference_of_row_magnitude"])


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_check_over_codes_still_finds_logits_that_are_off(dtype):
    from types import SimpleNamespace

    from metallix_b200.engine import cli
    rows = torch.randn((3, 50), generator=torch.Generator().manual_seed(0)).cuda()
    moved = torch.zeros_like(rows)
    moved[1, 7] = 0.25      # what the codes move a logit by

    def engine(logits):
        return SimpleNamespace(step=lambda entries: logits, check=lambda: None, release=lambda name: None)
    result = SimpleNamespace(input_ids=[1, 2], generated_ids=[3, 4, 5])
    absolute, relative = cli.VERIFY_BOUNDS[dtype]
    for times, within in ((0.0, True), (1.9, True), (2.2, False)):
        off = rows.clone()
        largest = rows[2].abs() if dtype == "float32" else rows[2].abs().amax()
        off[2] += times * 0.25 + (absolute + relative * largest) * (1.0 if times > 2 else 0.0)
        report = cli._verify_cache(engine(off), engine(rows), result, dtype, rows.cpu() - moved.cpu())
        assert report["logits_within_bound"] is within and abs(report["max_abs_logit_shift_of_codes"] - 0.25) < 1e-6
        assert cli._verify_cache(engine(off), engine(rows), result, dtype)["logits_within_bound"] is (times == 0.0)
