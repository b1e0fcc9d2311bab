"""Generation with keys and values held in 4 bits: against the plain implementation whose keys and values are packed the same way."""

import numpy as np
import pytest
import torch

import plain_llama as plain
from packed_plain import pack, quantize, values
from test_generate_gpu import engine_for, prompts_for
from tiny import page_size_of, tiny_model_dir

pytestmark = pytest.mark.gpu


def packed(x):
    code, word = quantize(x)
    return values(pack(code), word).to(x.dtype)


@pytest.fixture
def plain_packed(monkeypatch):
    """The plain implementation with every key (rotated) and value replaced by what 4 bits hold of it."""
    whole = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, *a, **o: whole(q, packed(k), packed(v), *a, **o))


@pytest.mark.parametrize("which, lengths, new, chunk", [("A", [5, 17, 33], 12, None), ("B", [1, 40, 100], 10, 24), ("C", [5, 70, 33], 12, None), ("D", [9, 40], 8, 16)])
def test_greedy_generation_equals_plain_float32(plain_packed, which, lengths, new, chunk):
    d = tiny_model_dir(which, 0.3)
    cfg, w = plain.read_config(d), plain.read_weights(d)
    prompts = prompts_for(cfg, lengths)
    eng = engine_for(d, "fp32", page_size=page_size_of(which), prefill_chunk=chunk, max_tokens_per_step=64, cache_bits=4)
    tokens, _, logits = eng.generate(prompts, tokens_to_generate=new, get_logits=True)
    for p, row, lg in zip(prompts, tokens.tolist(), logits):
        assert row == plain.greedy_generate(p, new, w, cfg)
        ref = plain.forward_logits(p + row[:-1], w, cfg)[len(p) - 1:]
        assert np.abs(lg.cpu().numpy() - ref.numpy()).max() <= 1e-4 * float(ref.abs().max())
    eng.engine.manager.check()
    assert all(eng.engine.manager.free_pages(g.name) == g.num_pages for g in eng.engine.groups)


@pytest.mark.parametrize("which, few", [("C", None), ("C", 0), ("D", 0)])
def test_bfloat16_recorded_steps_are_the_launched_ones(which, few, monkeypatch):
    """Decode steps replayed from recordings, prompts long enough for the unpacked form: the same tokens as launch by launch, and
    a cache of little more than a quarter of the bytes."""
    if few is not None:
        monkeypatch.setattr("yalis_b200.ops.packed.UNPACK_FEW", few)
    d = tiny_model_dir(which, 0.02)
    cfg = plain.read_config(d)
    prompts = prompts_for(cfg, [5, 90, 33, 64])
    got = []
    for graphs in (True, False):
        eng = engine_for(d, "bf16", page_size=16, cache_bits=4, use_graphs=graphs)
        got.append([eng.generate(prompts, tokens_to_generate=20)[0].tolist() for _ in range(2)])
        eng.engine.check_device_errors()
        small = eng.engine.storage.bytes
    assert got[0][0] == got[0][1] == got[1][0] == got[1][1]
    whole = engine_for(d, "bf16", page_size=16).engine.storage.bytes
    head = cfg["head_dim"]
    assert small * 2 * head * 2 == whole * (head + 4)


@pytest.mark.parametrize("few", [None, 0])
def test_bfloat16_follows_the_oracle(plain_packed, few, monkeypatch):
    """Every generated token is the oracle's best or within rounding of it."""
    if few is not None:
        monkeypatch.setattr("yalis_b200.ops.packed.UNPACK_FEW", few)
    d = tiny_model_dir("C", 0.02)
    cfg, w = plain.read_config(d), plain.read_weights(d)
    prompts = prompts_for(cfg, [5, 100, 33])
    tokens, _ = engine_for(d, "bf16", page_size=page_size_of("C"), cache_bits=4).generate(prompts, tokens_to_generate=16)
    for p, row in zip(prompts, tokens.tolist()):
        seq = list(p)
        for tok in row:
            ref = plain.forward_logits(seq, w, cfg)[-1]
            assert float(ref.max() - ref[tok]) <= 0.05 * float(ref.abs().max())
            seq.append(tok)


def test_caches_that_cannot_be_packed_are_refused():
    from yalis_b200.config.presets import preset
    from yalis_b200.engine.engine import Engine
    with pytest.raises(ValueError, match="4 bits"):
        Engine(config=preset("vepivik-tiny-A"), cache_bits=4, max_slots=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("parts, n, hs", [(1, 5, 64), (3, 5, 20), (1, 200, 64), (2, 200, 18), (2, 130, 128)])
def test_rotate_heads_gives_the_bits_of_the_cache_write(dtype, parts, n, hs):
    from yalis_b200.ops.elementwise import rope_kv_write, rotate_heads
    dev, nh, g, page = "cuda:0", 6, 2, 16
    gen = torch.Generator().manual_seed(hs + n)
    qkv = torch.randn(parts, n, (nh + 2 * g) * hs, generator=gen)
    qkv = qkv.to(dev) if parts > 1 else qkv[0].to(dev, dtype)
    positions = torch.arange(n, dtype=torch.int32, device=dev)
    reqs = torch.zeros(n, dtype=torch.int32, device=dev)
    reqs[-1] = -1
    inv = torch.rand(hs // 2, generator=gen).to(dev)
    pages = -(-n // page)
    k_pool, v_pool = (torch.zeros(pages, g, page, hs, dtype=dtype, device=dev) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    q = rope_kv_write(qkv, positions, reqs, inv, k_pool, v_pool, table, nh, g, hs, out_dtype=dtype)
    rows = rotate_heads(qkv, positions, reqs, inv, nh + 2 * g, hs, turned=nh + g, out_dtype=dtype)
    k, v = (p.permute(0, 2, 1, 3).reshape(-1, g * hs)[:n - 1] for p in (k_pool, v_pool))
    assert torch.equal(rows[:-1], torch.cat([q[:-1], k, v], 1))
    some = rotate_heads(qkv, positions, reqs, None, nh, hs, out_dtype=dtype)
    assert torch.equal(some[:-1], (qkv.sum(0) if parts > 1 and parts < 3 else qkv[0] + qkv[1] + qkv[2] if parts == 3 else qkv)[:-1, :nh * hs].to(dtype))


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("head_dim", [16, 64])
def test_windows_and_caches_that_two_layers_read(plain_packed, head_dim, graphs):
    """A layer over a window, whose pages are given back behind it, and one run twice over one cache, cut every way."""
    import tempfile

    import traces
    from test_toy_parts_gpu import plain_toy, setup_module, toy_config
    from yalis_b200.engine.engine import Engine
    from yalis_b200.engine.replay import Replayer
    from yalis_b200.weights.loader import write_random_model
    setup_module(None)
    c = toy_config(["window_attention", "attention"], [(0, None), (1, None), (1, 1)], window=20, head_dim=head_dim)
    with tempfile.TemporaryDirectory() as d:
        write_random_model(c, d, seed=5, std=0.2)
        w = plain.read_weights(d)
        g = torch.Generator().manual_seed(2)
        requests = {f"r{i}": torch.randint(0, c["vocab"], (n,), generator=g).tolist() for i, n in enumerate([150, 33, 97])}
        want = {rid: plain_toy(t, w, c).numpy() for rid, t in requests.items()}
        for build in (traces.whole, traces.tail_decoded, traces.portions, traces.mixed):
            steps = traces.number(build(requests))
            tokens = traces.peak_tokens(steps)
            rep = Replayer(d, "float32", tokens, page_size=8, graphs=graphs,
                           engine=Engine(d, dtype="float32", page_size=8, num_pages=-(-tokens // 64) * 8, max_slots=4, cache_bits=4))
            assert sorted(x.name for x in rep.engine.groups) == ["kv_all", "kv_window_20"]
            out = {}
            for s in steps:
                r = rep.run_step(s)
                if r is not None:
                    out[s["step"]] = r
            got = traces.collect(steps, out, c["vocab"])
            for rid in want:
                assert np.abs(got[rid] - want[rid]).max() <= 1e-4 * np.abs(want[rid]).max(), (build.__name__, rid)
            rep.engine.manager.check()


def test_position_encodings_that_store_by_themselves_are_refused():
    import tempfile

    from test_toy_parts_gpu import setup_module, toy_config
    from yalis_b200.engine.engine import Engine
    from yalis_b200.weights.loader import write_random_model
    setup_module(None)
    c = toy_config(["attention"], [(0, None)], positions=["decay"])
    with tempfile.TemporaryDirectory() as d:
        write_random_model(c, d, seed=5, std=0.2)
        with pytest.raises(ValueError, match="4 bits"):
            Engine(d, dtype="float32", page_size=8, num_pages=8, max_slots=2, cache_bits=4)
