"""The 4-bit cache without a GPU: the layout the plain implementation keeps, and what the wrappers refuse."""
import pytest
import torch

from tests.plain import kv4_plain as plain
from vllm_oxide_b200 import kernels
from vllm_oxide_b200.errors import KernelError, ShapeError


@pytest.mark.parametrize("hd,page", [(16, 8), (48, 24), (64, 16), (128, 16), (256, 8), (80, 40)])
def test_packing_all_at_once_and_one_by_one_make_the_same_bytes(hd, page):
    g, G = torch.Generator().manual_seed(hd), 2
    k, v = torch.randn(2 * page, G, hd, generator=g), torch.randn(2 * page, G, hd, generator=g)
    cache, kk, vv = plain.pack(k, v, page)
    assert cache.shape == (2, G, page, kernels.kv4_width(hd))
    other = torch.full_like(cache, 255)
    for which, x, held in ((0, k, kk), (1, v, vv)):
        n, s, m = plain.quantise(x)
        for t in range(2 * page):
            for h in range(G):
                plain.write(other, t // page, h, t % page, which, n[t, h], s[t, h], m[t, h])
                assert torch.equal(plain.read(cache, t // page, h, t % page, which, hd), held[t, h])
    assert torch.equal(cache, other)
    # a code is at most half a step off, plus what rounding s and m to bfloat16 (2^-8 each) moves
    n, s, m = plain.quantise(k)
    off = (kk - k.double()).abs()
    assert (off <= 0.5 * s.double()[..., None] * (1 + 1e-6) + 2.0 ** -8 * (15 * s.abs() + m.abs()).double()[..., None]).all()


@pytest.fixture
def no_gpu(monkeypatch):
    """Shapes, types and strides are checked before devices: what does not fit is refused wherever the tensors are."""
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda d: type("P", (), {"multi_processor_count": 148})())


def _append_args(**change):
    H, G, hd, T = 4, 2, 32, 3
    a = dict(q=torch.zeros(T, H * hd), k=torch.zeros(T, G * hd), v=torch.zeros(T, G * hd), positions=torch.zeros(T, dtype=torch.int32),
             slots=torch.zeros(T, dtype=torch.int32), inv_freq=torch.ones(hd // 2), cache=torch.zeros(5, G, 16, 40, dtype=torch.uint8),
             num_heads=H, num_kv_heads=G, head_dim=hd)
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(cache=torch.zeros(5, 2, 16, 40)), dict(cache=torch.zeros(5, 2, 16, 32, dtype=torch.uint8)),
    dict(cache=torch.zeros(5, 2, 12, 40, dtype=torch.uint8)), dict(cache=torch.zeros(5, 3, 16, 40, dtype=torch.uint8)),
    dict(cache=torch.zeros(0, 2, 16, 40, dtype=torch.uint8)), dict(cache=torch.zeros(5, 2, 16, 80, dtype=torch.uint8)[..., ::2]),
    dict(cache=torch.zeros(5 * 2 * 16 * 40 + 1, dtype=torch.uint8)[1:].view(5, 2, 16, 40)),
    dict(q=torch.zeros(3, 127)), dict(k=torch.zeros(2, 64)), dict(v=torch.zeros(3, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 256)[:, ::2]), dict(q=torch.zeros(3, 128, dtype=torch.float16), k=torch.zeros(3, 64, dtype=torch.float16),
                                               v=torch.zeros(3, 64, dtype=torch.float16)),
    dict(positions=torch.zeros(2, dtype=torch.int32)), dict(positions=torch.zeros(3, dtype=torch.int64)),
    dict(slots=torch.zeros(3)), dict(inv_freq=torch.ones(32)), dict(inv_freq=torch.ones(16).double()), dict(num_heads=3, q=torch.zeros(3, 96)),
    dict(q_out=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(q_out=torch.zeros(4, 128)),
    dict(head_dim=24, q=torch.zeros(3, 96), k=torch.zeros(3, 48), v=torch.zeros(3, 48), inv_freq=torch.ones(12))])
def test_append_refuses(no_gpu, change):
    with pytest.raises(ShapeError):
        kernels.kv4_append(**_append_args(**change))


def _attn_args(**change):
    H, G, hd, S = 4, 2, 32, 3
    a = dict(q=torch.zeros(S, H * hd), out=torch.zeros(S, H * hd), cache=torch.zeros(5, G, 16, 40, dtype=torch.uint8),
             block_tables=torch.zeros(S, 2, dtype=torch.int32), num_heads=H, num_kv_heads=G, head_dim=hd, scale=1.0)
    a.update(change)
    return a


ATTN = [dict(q=torch.zeros(3, 120)), dict(out=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(out=torch.zeros(2, 128)),
        dict(cache=torch.zeros(5, 2, 16, 36, dtype=torch.uint8)), dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)),
        dict(block_tables=torch.zeros(3, 2)), dict(window=-1), dict(out=torch.zeros(3, 256)[:, ::2]),
        dict(q=torch.zeros(3, 128).half(), out=torch.zeros(3, 128).half())]


@pytest.mark.parametrize("change", ATTN + [dict(positions=torch.zeros(2, dtype=torch.int32)),
                                           dict(scratch=(2, 4, 2, 32)), dict(scratch=(3, 8, 2, 32)), dict(scratch=(3, 4, 2, 64))])
def test_decode_refuses(no_gpu, change):
    a = _attn_args(positions=torch.zeros(3, dtype=torch.int32), scratch=(3, 4, 2, 32))
    a.update(change)
    a["scratch"] = kernels.kv4_scratch(*a["scratch"], "cpu")
    with pytest.raises(ShapeError):
        kernels.attn_decode_kv4(**a)


@pytest.mark.parametrize("change", ATTN + [dict(seq_starts=torch.zeros(3, dtype=torch.int32)), dict(context_lens=torch.zeros(3))])
def test_portions_refuse(no_gpu, change):
    a = _attn_args(seq_starts=torch.zeros(4, dtype=torch.int32), context_lens=torch.zeros(3, dtype=torch.int32), num_seqs=3, max_new=1)
    a.update(change)
    with pytest.raises(ShapeError):
        kernels.attn_prefill_kv4(**a)


def test_there_is_no_cpu_path(no_gpu):
    """Calls that fit, on the CPU."""
    c = torch.zeros(2, 1, 8, kernels.kv4_width(16), dtype=torch.uint8)
    x, i, t = torch.zeros(1, 16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: kernels.kv4_append(x, x, x, i, i, None, c, 1, 1, 16), lambda: kernels.kv4_read(c, i, x, x, 1, 16),
                 lambda: kernels.attn_decode_kv4(x, x, c, t, i, 1, 1, 16, 1.0, scratch=kernels.kv4_scratch(1, 1, 1, 16, "cpu")),
                 lambda: kernels.attn_prefill_kv4(x, x, c, t, torch.zeros(2, dtype=torch.int32), i, 1, 1, 1, 1, 16, 1.0),
                 lambda: kernels.kv4_append(**_append_args()), lambda: kernels.kv4_append(**_append_args(q_out=torch.zeros(3, 128), slots=None)),
                 lambda: kernels.kv4_append(**_append_args(q=torch.zeros(3, 300)[:, 9:137], inv_freq=None))):
        with pytest.raises(KernelError, match="no CPU path"):
            call()


def test_scratch_refuses(no_gpu):
    for bad in ((-1, 4, 2, 32), (1, 3, 2, 32), (1, 4, 2, 24), (1, 4, 0, 32)):
        with pytest.raises(ShapeError):
            kernels.kv4_scratch(*bad, "cpu")


def test_engine_config_takes_four_or_none():
    from vllm_oxide_b200.config import EngineConfig
    from vllm_oxide_b200.errors import ConfigError
    assert EngineConfig().cache_bits is None and EngineConfig(cache_bits=4).cache_bits == 4
    for bad in (3, 8, 16, "4", 4.5, 4.0, True, 0):
        with pytest.raises(ConfigError, match="cache_bits"):
            EngineConfig(cache_bits=bad)


def test_architectures_say_what_they_cache():
    from vllm_oxide_b200 import models  # noqa: F401
    from vllm_oxide_b200.config import architecture_for, known_architectures
    assert [a for a in known_architectures() if 4 in architecture_for({"architectures": [a]}).cache_bits] == ["LlamaForCausalLM"]


@pytest.mark.parametrize("odd", [5, None, "q", torch.zeros(3, 128).to_sparse(), torch.zeros(1, 1, 1, 3, 128), torch.zeros(3, 128, dtype=torch.complex64),
                                 torch.zeros((), dtype=torch.float32), torch.zeros(0)])
def test_what_is_no_tensor_with_rows_is_refused(no_gpu, odd):
    with pytest.raises(ShapeError):
        kernels.kv4_append(**_append_args(q=odd))
    with pytest.raises(ShapeError):
        kernels.attn_prefill_kv4(**_attn_args(q=odd, seq_starts=torch.zeros(4, dtype=torch.int32), context_lens=torch.zeros(3, dtype=torch.int32),
                                              num_seqs=3, max_new=1))
