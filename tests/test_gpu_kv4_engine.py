"""The engine on a 4-bit cache: traces against the plain implementation that reads the keys and values which the engine holds, generation
with and without graphs, the command line, graphs and streams around the kernels, and what is refused."""
import json
import os
import subprocess
import sys

import pytest
import torch

from tests.plain import kv4_plain, llama_plain as plain
from tests.test_gpu_replay import run_trace
from tests.util import TINY, TOL, make_model_dir, max_rel_diff, random_tokens

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from vllm_oxide_b200 import kernels
    kernels.gemm_sm100_check()


def session(model_dir, dtype, page, pages, **kw):
    from vllm_oxide_b200.config import EngineConfig
    from vllm_oxide_b200.engine import ModelRunner
    from vllm_oxide_b200.replay.trace import TraceSession
    args = dict(max_batch_tokens=pages * page, max_seqs=8, max_model_len=pages * page, block_size=page, num_pages=pages, dtype=dtype,
                cuda_graphs=False, cache_bits=4)
    args.update(kw)
    return TraceSession(ModelRunner.from_dir(model_dir, EngineConfig(**args)))


def cached(sess, name, cfg):
    """Per layer the keys and values [T, heads * hd] that the engine holds of a request, float64 on the CPU."""
    from vllm_oxide_b200 import kernels
    r = sess.runner
    rid, page = sess.ids[name], r.engine.block_size
    T = r.manager.length(rid)
    table = r.manager.block_table(rid, 0)
    slots = torch.tensor([table[t // page] * page + t % page for t in range(T)], dtype=torch.int32, device=DEV)
    G, hd = cfg.num_key_value_heads, cfg.head_dim
    got = []
    for layer in range(cfg.num_hidden_layers):
        k, v = (torch.empty(T, G * hd, device=DEV) for _ in range(2))
        kernels.kv4_read(r.pools.kv[layer][0], slots, k, v, G, hd)
        got.append((k.double().cpu(), v.double().cpu()))
    return got


def plain_logits(model_dir, tokens, held, cfg, dtype, monkeypatch):
    """Logits of the plain implementation whose layers read the keys and values `held`, each of which must be the layer's own in 4 bits:
    at most half a step and the engine's own rounding off."""
    layer = [0]
    full = plain.causal_attention
    # what the engine's keys and values may be off by before they are quantised: as its logits may be (TOL)
    own = TOL[dtype]

    def attention(q, k, v, H, KV, hd, window=None, scale=None):
        hk, hv = held[layer[0]]
        layer[0] += 1
        for x, h in ((k, hk), (v, hv)):
            x, h = x.view(-1, KV, hd), h.view(-1, KV, hd)
            n, s, m = kv4_plain.quantise(x.float())
            # s and m in bfloat16: 2^-8 of them; a step more where a code's neighbour was taken
            room = 0.5 * s.double().abs() + 2.0 ** -8 * (15 * s.abs() + m.abs()).double() + 2 * own * x.abs().amax()
            assert ((h - x).abs() <= room[..., None] * (1 + 1e-5)).all()
        return full(q, hk, hv, H, KV, hd, window, scale)
    monkeypatch.setattr(plain, "causal_attention", attention)
    pc, pt = plain.load_model(model_dir)
    out = plain.forward(pc, pt, list(tokens))
    monkeypatch.undo()
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["B", "C", "D", "HD128"])
def test_a_trace_of_portions_and_single_tokens(tmp_path_factory, name, dtype, monkeypatch):
    cfg, _, page = TINY[name]
    d = make_model_dir(tmp_path_factory.getbasetemp(), name)
    sess = session(d, dtype, page, 256 // page)
    toks = {"a": random_tokens(75, cfg.vocab_size, 1), "b": random_tokens(41, cfg.vocab_size, 2)}
    steps = [{"entries": [{"id": "a", "tokens": toks["a"][:33], "want": [0, 32]}]},
             {"entries": [{"id": "a", "tokens": toks["a"][33:34], "want": [0]}, {"id": "b", "tokens": toks["b"][:35], "want": [4, 34]}]},
             {"entries": [{"id": "a", "tokens": toks["a"][34:70], "want": [35]}, {"id": "b", "tokens": toks["b"][35:36], "want": [0]}]}]
    for i in range(5):
        steps.append({"entries": [{"id": "a", "tokens": [toks["a"][70 + i]], "want": [0]}, {"id": "b", "tokens": [toks["b"][36 + i]], "want": [0]}]})
    got = run_trace(sess, [{"step": i, "end": [], **s} for i, s in enumerate(steps)])
    assert len(got) == 2 + 3 + 2 + 10
    for who in ("a", "b"):
        ref = plain_logits(d, toks[who], cached(sess, who, cfg), cfg, dtype, monkeypatch)
        for (n, p), row in got.items():
            if n == who:
                assert max_rel_diff(row, ref[p]) <= TOL[dtype], (who, p)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_with_and_without_graphs(tmp_path_factory, dtype):
    from vllm_oxide_b200.engine import LLM
    from vllm_oxide_b200.sampling import SamplingParams
    cfg, _, page = TINY["D"]
    d = make_model_dir(tmp_path_factory.getbasetemp(), "D")
    prompts = [random_tokens(n, cfg.vocab_size, n) for n in (150, 9, 70, 33)]
    outs = []
    for kw in (dict(), dict(cuda_graphs=False, run_ahead=False), dict(pdl=False)):
        llm = LLM(d, dtype=dtype, cache_bits=4, max_batch_tokens=128, max_seqs=4, max_model_len=256, block_size=page, num_pages=64, **kw)
        p = SamplingParams(max_new_tokens=20, stop_token_ids=())
        first = [o.token_ids for o in llm.generate(prompts, p)]
        assert [o.token_ids for o in llm.generate(prompts, p)] == first
        if not kw:
            assert llm.stats["graph_steps"] > 0 and llm.stats["ahead_steps"] > 0
            # one layer's page of 16 tokens: 64 + 8 bytes a token and kv head
            assert llm.runner.pools.bytes_per_token() == cfg.num_hidden_layers * cfg.num_key_value_heads * 72
        outs.append(first)
    assert outs[0] == outs[1] == outs[2]


def test_pages_run_out_and_requests_are_taken_up_again(tmp_path_factory):
    """A pool that cannot hold all requests at once: preempted requests compute their tokens anew, in pages that others used."""
    from vllm_oxide_b200.engine import LLM
    from vllm_oxide_b200.sampling import SamplingParams
    cfg, _, page = TINY["D"]
    d = make_model_dir(tmp_path_factory.getbasetemp(), "D")
    prompts = [random_tokens(n, cfg.vocab_size, n) for n in (60, 50, 61, 40)]
    p = SamplingParams(max_new_tokens=40, stop_token_ids=())
    roomy = LLM(d, dtype="float32", cache_bits=4, max_batch_tokens=128, max_seqs=4, max_model_len=128, block_size=page, num_pages=64)
    tight = LLM(d, dtype="float32", cache_bits=4, max_batch_tokens=128, max_seqs=4, max_model_len=128, block_size=page, num_pages=18)
    want = [o.token_ids for o in roomy.generate(prompts, p)]
    got = tight.generate(prompts, p)
    assert sum(o.preemptions for o in got) > 0
    assert all(len(o.token_ids) == 40 for o in got)
    assert [o.token_ids[:8] for o in got] == [w[:8] for w in want]


def test_the_attention_part_in_a_window_and_with_a_cache_of_another_layer(tmp_path):
    """`Attention(cache_bits=4)` put together by hand: a windowed layer, and one that reads the cache that the first wrote."""
    from vllm_oxide_b200.cache.pools import CachePools
    from vllm_oxide_b200.parts import Attention, LayerCall, Rotary, StepContext, Workspace
    H, G, hd, hidden, n, page, window = 4, 2, 64, 96, 50, 8, 21
    g = torch.Generator().manual_seed(4)

    def w(o, i):
        return 0.1 * torch.randn(o, i, generator=g)
    rot = Rotary(hd, 10000.0, None, DEV)
    wq, wk, wv, wo, wq2 = w(H * hd, hidden), w(G * hd, hidden), w(G * hd, hidden), w(hidden, H * hd), w(H * hd, hidden)
    kw = dict(position=rot, window=window, dtype=torch.float32, device=DEV, cache_bits=4)
    first, second = Attention(wq, wk, wv, wo, H, G, hd, **kw), Attention(wq2, None, None, wo, H, G, hd, **kw)
    spec = type("Spec", (), dict(blocks=[type("B", (), dict(mixer=m))() for m in (first, second)], embedding=None,
                                 schedule=[LayerCall(0, 0, True), LayerCall(1, 0, False)]))()
    pools = CachePools(spec, page, 2, torch.float32, DEV, num_pages=16)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.randperm(16, generator=g)[:7]
    x = torch.randn(n, hidden, generator=g)
    outs = [[], []]
    for a, b in ((0, 30), (30, 49), (49, 50)):
        T = b - a
        ws = Workspace(1 << 22, DEV)
        pos = torch.arange(a, b)
        ctx = StepContext(rows=T, seqs=1, dtype=torch.float32, tokens=torch.zeros(T, **i32), positions=pos.int().to(DEV), row_seq=torch.zeros(T, **i32),
                          seq_starts=torch.tensor([0, T], **i32), context_lens=torch.tensor([a], **i32), seq_lens=torch.tensor([b], **i32),
                          state_slots=torch.zeros(1, **i32), logit_rows=torch.zeros(1, **i32),
                          slot_mapping=[(table[pos // page] * page + pos % page).int().to(DEV)], block_tables=[table.int().to(DEV).view(1, 7)],
                          workspace=ws, max_new=T, decode_only=T == 1)
        for k, (m, write) in enumerate(((first, True), (second, False))):
            outs[k].append(m.forward(x[a:b].to(DEV), ctx, pools.layer_cache(0, write), None).cpu().double().clone())
    xd = x.double()
    f = rot.inv_freq.cpu()
    k = kv4_plain.rotate((xd @ wk.double().t()).view(n, G, hd), torch.arange(n), f).float()
    kk, vv = (kv4_plain.values(*kv4_plain.quantise(y)) for y in (k, (xd @ wv.double().t()).float().view(n, G, hd)))
    for got, wqi in zip(outs, (wq, wq2)):
        q = kv4_plain.rotate((xd @ wqi.double().t()).view(n, H, hd), torch.arange(n), f)
        ref, _, _ = kv4_plain.attend(q, kk, vv, torch.arange(n), hd ** -0.5, window)
        ref = ref.reshape(n, H * hd) @ wo.double().t()
        # a code at a border may fall to its neighbour's side in one of 50 x 128 numbers: one step (a tenth of a number's size) of
        # one of some 20 keys, through a projection of 256: below 2e-3 of the largest result; 2e-5 without one
        assert max_rel_diff(torch.cat(got), ref) <= 2e-3


def test_captured_and_replayed_with_new_contents_on_another_stream():
    """One graph of append, single-token attention and attention of a portion, replayed with other rows, lengths and pages in the same buffers;
    two graphs that share a scratch, one behind the other."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page, pages, S = 8, 2, 64, 16, 40, 3
    g = torch.Generator().manual_seed(9)
    i32 = dict(dtype=torch.int32, device=DEV)
    cache = kv4_plain.pack(torch.randn(pages * page, G, hd, generator=g), torch.randn(pages * page, G, hd, generator=g), page)[0].to(DEV)
    f = torch.tensor([1e4 ** (-2 * i / hd) for i in range(hd // 2)], device=DEV)
    qkv = torch.zeros(S, (H + 2 * G) * hd, dtype=torch.bfloat16, device=DEV)
    pos, slots, tab = torch.zeros(S, **i32), torch.zeros(S, **i32), torch.zeros(S, 13, **i32)
    starts, ctxs = torch.tensor([0, 1, 2, 3], **i32), torch.zeros(S, **i32)
    q, k, v = qkv.split((H * hd, G * hd, G * hd), dim=1)
    qr, o1, o2 = (torch.zeros(S, H * hd, dtype=torch.bfloat16, device=DEV) for _ in range(3))
    scratch = kernels.kv4_scratch(S, H, G, hd, DEV)

    def step(c):
        kernels.kv4_append(q, k, v, pos, slots, f, c, H, G, hd, q_out=qr)
        kernels.attn_decode_kv4(qr, o1, c, tab, pos, H, G, hd, hd ** -0.5, scratch=scratch)
        kernels.attn_prefill_kv4(qr, o2, c, tab, starts, ctxs, S, 1, H, G, hd, hd ** -0.5)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(cache.clone())
        side.synchronize()
        work = cache.clone()
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                step(work)
            graphs.append(gr)
        for trial, lens in enumerate(([1, 2, 200], [17, 130, 64], [208, 5, 33])):
            order = torch.randperm(pages, generator=g)
            tab.copy_(order[:39].view(3, 13))
            pos.copy_(torch.tensor(lens) - 1)
            ctxs.copy_(torch.tensor(lens) - 1)
            slots.copy_(torch.tensor([int(order[13 * s + (n - 1) // page]) * page + (n - 1) % page for s, n in enumerate(lens)]))
            qkv.copy_(torch.randn(S, (H + 2 * G) * hd, generator=g))
            work.copy_(cache)
            for gr in graphs:
                o1.zero_(), o2.zero_()
                gr.replay()
            side.synchronize()
            got = [x.clone() for x in (qr, o1, o2, work)]
            work.copy_(cache)
            step(work)
            side.synchronize()
            # (tokens written twice are the same bytes; a call does not depend on what ran before it)
            for a, b in zip(got, (qr, o1, o2, work)):
                assert torch.equal(a, b), trial
            # the two attentions agree to their roundings: 2^-8 of the result and of the probabilities, keys and values as numbers of bfloat16
            assert (o1.float() - o2.float()).abs().max() <= 8 * 2.0 ** -8 * o1.float().abs().max()
    assert int(scratch.arrived.abs().sum()) == 0


def test_the_command_line_and_trace_run(tmp_path):
    from tests.util import TINY_B
    from vllm_oxide_b200.weights import write_random_model
    d = str(tmp_path / "m")
    write_random_model(d, TINY_B, 3, std=0.08)
    args = [sys.executable, "-m", "vllm_oxide_b200", "generate", d, "--prompt-ids", "5,17,3", "--max-new", "6", "--max-model-len", "64",
            "--num-pages", "16", "--block-size", "8", "--cache-bits"]
    ok = subprocess.run(args + ["4"], capture_output=True, text=True, cwd=ROOT)
    assert ok.returncode == 0 and len(ok.stdout.split()) <= 6 and ok.stdout.split(), ok.stderr[-2000:]
    bad = subprocess.run(args + ["3"], capture_output=True, text=True, cwd=ROOT)
    assert bad.returncode == 1 and "cache_bits" in bad.stderr and "Traceback" not in bad.stderr
    msg = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3, 9], "want": [3]}], "end": ["a"]})
    run = subprocess.run([os.path.join(ROOT, "bin", "trace_run"), "--model", d, "--dtype", "float32", "--out", str(tmp_path / "o"), "--max-tokens", "32",
                          "--cache-bits", "4"], input=msg + "\n", capture_output=True, text=True, cwd=ROOT)
    assert run.returncode == 0 and run.stdout.strip() == "done 0", run.stderr[-2000:]
    assert os.path.getsize(str(tmp_path / "o" / "0.f32")) == 4 * TINY_B.vocab_size


def test_an_architecture_that_does_not_name_it_is_refused():
    from tests.test_rotepel_config import _dict as rotepel
    from vllm_oxide_b200.config import EngineConfig, architecture_for
    from vllm_oxide_b200.engine import ModelRunner
    from vllm_oxide_b200.errors import ConfigError
    arch = architecture_for(rotepel())
    with pytest.raises(ConfigError, match="4 bits"):
        ModelRunner(arch.config_cls.from_dict(rotepel()), {}, EngineConfig(cache_bits=4), arch)
