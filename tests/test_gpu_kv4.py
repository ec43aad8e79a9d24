"""The cache in 4 bits: appending to it with the rotary positions applied on the way, reading it back, attention over it for single
tokens and for portions, against the definition in 64 bits (tests/plain/kv4_plain.py)."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}            # half a step, relative to the value


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from vllm_oxide_b200 import kernels
    kernels.gemm_sm100_check()


def freq(hd, base=500000.0):
    return torch.tensor([base ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=F32)


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ append, read back
def append_case(T, H, G, hd, page, dtype, seed, start=0, rope=True, strided=True, extra=None):
    from vllm_oxide_b200 import kernels
    g = gen(seed)
    pages = -(-T // page) + 3
    qkv = torch.randn(T, (H + 2 * G) * hd + (8 if strided else 0), generator=g)
    if extra is not None:
        extra(qkv)
    qkv = qkv.to(dtype)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    positions = (torch.arange(T) * 3 + start).int()
    f = freq(hd) if rope else None
    before = torch.randint(0, 256, (pages, G, page, plain.width(hd)), generator=g, dtype=torch.uint8)
    dev = qkv.to(DEV)
    q, k, v = dev[:, :H * hd], dev[:, H * hd:(H + G) * hd], dev[:, (H + G) * hd:(H + 2 * G) * hd]
    cache = before.to(DEV)
    q_out = torch.empty(T, H * hd, dtype=dtype, device=DEV)
    kernels.kv4_append(q, k, v, positions.to(DEV), slots.to(DEV), f.to(DEV) if rope else None, cache, H, G, hd, q_out=q_out)
    torch.cuda.synchronize()
    return qkv, slots, positions, f, before, cache, q_out, dev


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,G,hd,page,start", [(1, 4, 2, 64, 16, 0), (3, 3, 3, 16, 8, 5), (37, 6, 3, 48, 24, 100), (130, 8, 1, 128, 16, 130000),
                                                 (19, 5, 5, 80, 40, 7), (9, 2, 1, 256, 8, 9999), (5, 6, 2, 96, 64, 1), (700, 4, 2, 64, 16, 3)])
def test_append_writes_the_definitions_bytes(T, H, G, hd, page, start, dtype):
    qkv, slots, positions, f, before, cache, q_out, dev = append_case(T, H, G, hd, page, dtype, 7 * T + hd, start)
    x = qkv[:, :(H + 2 * G) * hd].view(T, H + 2 * G, hd)
    want = before.clone()
    k = plain.rotate(x[:, H:H + G], positions, f).float()
    for which, y in ((0, k), (1, x[:, H + G:].float())):
        n, s, m = plain.quantise(y)
        for t in range(T):
            for h in range(G):
                plain.write(want, int(slots[t]) // page, h, int(slots[t]) % page, which, n[t, h], s[t, h], m[t, h])
    # codes are decisions: a byte that differs stands for a number a whole step off. The rotation is taken in 64 bits on both sides
    # and rounded to 32 once, so a rotated key can differ by one 32-bit step only where the two 64-bit sines do; none may reach a code
    assert torch.equal(cache.cpu(), want)
    # q: the exact value rounded to 32 bits and to its type. Where the two products cancel, what is left shows the angle's own rounding:
    # its share of pi, rounded to 64 bits (2^-53 of it), and the 64-bit sine and cosine (2^-52) move a number by less than
    # (angle + 2) * 2^-52 * (|x_i| + |x_(i + hd/2)|)
    ref = plain.rotate(x[:, :H], positions, f).reshape(T, H * hd)
    turned = (positions.double().max() + 2) * 2.0 ** -52 * 2 * x.abs().double().max()
    if dtype == BF16:
        # q of bfloat16 is turned in 32 bits: sine, cosine, two products and a sum, each rounded by at most 2^-24 of numbers up to |x_i| + |x_(i + hd/2)|
        turned += 4 * 2.0 ** -24 * 2 * x.abs().double().max()
    assert ((q_out.cpu().double() - ref).abs() <= (HALF[dtype] + 2.0 ** -24) * ref.abs() + turned).all()
    assert torch.equal(dev.cpu(), qkv)                   # what came in is left as it was


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd,page", [(64, 16), (48, 24), (256, 8), (128, 64)])
def test_read_gives_what_the_bytes_stand_for(hd, page, dtype):
    from vllm_oxide_b200 import kernels
    g, G, pages, T = gen(hd), 3, 5, 41
    k, v = torch.randn(pages * page, G, hd, generator=g), 100 * torch.randn(pages * page, G, hd, generator=g)
    cache, kk, vv = plain.pack(k, v, page)
    slots = torch.randint(0, pages * page, (T,), generator=g).int()
    slots[3], slots[4] = -1, pages * page
    ko, vo = (torch.full((T, G * hd + 3), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    kernels.kv4_read(cache.to(DEV), slots.to(DEV), ko[:, :G * hd], vo[:, :G * hd], G, hd)
    for got, ref in ((ko.cpu(), kk), (vo.cpu(), vv)):
        assert (got[:, G * hd:] == 7).all()
        got, ref = got[:, :G * hd].double(), ref[slots.long().clamp(0, pages * page - 1)].reshape(T, G * hd).clone()
        assert (got[3] == 0).all() and got[4].isnan().all()
        ref[3], ref[4], got[4] = 0, 0, 0
        # m + s n: s n is exact in 32 bits, one rounding of the sum, one to the output's type
        assert ((got - ref).abs() <= (HALF[dtype] + 2.0 ** -24) * ref.abs()).all()


def test_append_in_place_without_rotation_and_without_slots():
    from vllm_oxide_b200 import kernels
    H, G, hd, page, T = 4, 2, 64, 16, 6
    qkv, slots, positions, f, before, cache, q_out, _ = append_case(T, H, G, hd, page, BF16, 3, rope=False)
    assert torch.equal(q_out.cpu(), qkv[:, :H * hd])
    ko, vo = (torch.empty(T, G * hd, dtype=F32, device=DEV) for _ in range(2))
    kernels.kv4_read(cache, slots.to(DEV), ko, vo, G, hd)
    n, s, m = plain.quantise(qkv[:, H * hd:(H + G) * hd].float().view(T, G, hd))
    assert torch.equal(ko.cpu(), plain.values(n, s, m).float().view(T, G * hd))
    # in place, no slots: q turns, the cache stays
    q = qkv.to(DEV)
    kept = cache.clone()
    a = [q[:, :H * hd], q[:, H * hd:(H + G) * hd], q[:, (H + G) * hd:(H + 2 * G) * hd]]
    kernels.kv4_append(*a, positions.to(DEV), None, freq(hd).to(DEV), cache, H, G, hd)
    ref = plain.rotate(qkv[:, :H * hd].view(T, H, hd), positions, freq(hd)).reshape(T, H * hd)
    # turned in 32 bits: see above
    assert ((a[0].cpu().double() - ref).abs() <= HALF[BF16] * ref.abs() + 8 * 2.0 ** -24 * qkv.abs().double().max()).all()
    assert torch.equal(cache, kept)
    # slots behind the pool and negative ones are not kept either
    bad = torch.tensor([-1, cache.shape[0] * page, -7, 2 ** 31 - 1, -1, cache.shape[0] * page + 5], dtype=torch.int32, device=DEV)
    kernels.kv4_append(*a, positions.to(DEV), bad, None, cache, H, G, hd)
    assert torch.equal(cache, kept)
    kernels.kv4_append(*[t[:0] for t in a], positions[:0].to(DEV), bad[:0], None, cache, H, G, hd)     # no tokens
    assert torch.equal(cache, kept)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_keeps_odd_vectors(dtype):
    """Constant vectors, zeros, numbers next to the type's largest and smallest, infinities and NaN."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page, T = 1, 1, 64, 8, 9

    def extra(x):
        k = x[:, hd:2 * hd]
        k[0] = 0.0
        k[1] = 3.25
        k[2] = -1e30
        k[2, 5] = 1e30
        k[3, 7] = math.inf
        k[4, 9] = -math.inf
        k[5, 11] = math.nan
        k[6] = 1e-39
        k[7] = -3.3e38
        k[7, 0] = 3.3e38
        k[8] *= 1e-36
    qkv, slots, positions, f, before, cache, q_out, _ = append_case(T, H, G, hd, page, dtype, 5, rope=False, extra=extra)
    ko, vo = (torch.empty(T, hd, dtype=F32, device=DEV) for _ in range(2))
    kernels.kv4_read(cache, slots.to(DEV), ko, vo, G, hd)
    n, s, m = plain.quantise(qkv[:, hd:2 * hd].float())
    want = plain.values(n, s, m).float()
    got = ko.cpu()
    for t in range(T):
        if t in (3, 4, 5):
            assert got[t].isnan().all(), t
        else:
            assert torch.equal(got[t], want[t]), t
    assert (got[0] == 0).all() and (got[1] == 3.25).all()


# ------------------------------------------------------------------------------------------------ attention
def paged(lens, G, hd, page, seed, k_scale=1.0, garbage=True):
    """Requests of these lengths in pages strewn over a pool -> (cache, block tables on the device, keys and values per request).
    What the pool holds beside them, the rest of their last pages included, is NaN in scale and minimum and any codes."""
    g = gen(seed)
    W = plain.width(hd)
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g)
    cache = torch.randint(0, 256, (total, G, page, W), generator=g, dtype=torch.uint8)
    C = -(-hd // 32)
    if garbage:
        cache.view(total, G, page // 8, 8 * W)[..., 256 * C:] = 255                 # NaN in bfloat16
    tables = torch.full((len(lens), max(max(need), 1) + 2), -1, dtype=torch.int32)
    at, keys, vals = 0, [], []
    for s, n in enumerate(lens):
        L = need[s] * page
        k = k_scale * torch.randn(L, G, hd, generator=g) * (1 + 3 * (torch.rand(G, hd, generator=g) < 0.05))
        v = torch.randn(L, G, hd, generator=g) * (0.2 + torch.rand(L, G, 1, generator=g))
        if L:
            k[n:], v[n:] = math.nan, math.nan
            packed, kk, vv = plain.pack(k, v, page)
            pages = order[at:at + need[s]]
            cache[pages] = packed
            tables[s, :need[s]] = pages.int()
        else:
            kk, vv = k.double(), v.double()
        at += need[s]
        keys.append(kk[:n])
        vals.append(vv[:n])
    return cache.to(DEV), tables.to(DEV), keys, vals


def tolerance(ref, size, mag, vmax, dtype):
    """How far a row may be off. 32 bits: the scores' products and sums (at most 2^-24 a step, some hundred steps, on numbers that
    add up to `size`), twice (numerator and denominator), and the sums of the values. bfloat16: q as given; the kernels that make numbers of
    the codes round them to bfloat16 (2^-8 of every key: 2^-8 `size` on a score, twice; 2^-8 of every value) and the probabilities too
    (2^-8 of `mag`, twice); the result 2^-8."""
    if dtype == F32:
        return 2.0 ** -24 * ref.abs() + (2 * 64 * 2.0 ** -24 * size + 512 * 2.0 ** -24) * (mag + ref.abs()) + 1e-30
    return 2.0 ** -8 * ref.abs() + (2 * 2.0 ** -8 * size + 3 * 2.0 ** -8) * (mag + ref.abs()) + 1e-30


DECODE = [  # lengths, heads, kv heads, head size, page, window
    ([1], 4, 2, 64, 16, 0), ([2, 1, 3], 4, 4, 64, 8, 0), ([100], 8, 2, 64, 16, 0), ([129, 64, 65, 63], 6, 2, 128, 16, 0),
    ([700, 1, 33, 256], 8, 1, 128, 24, 0), ([515], 16, 1, 64, 64, 0), ([300, 31], 20, 1, 80, 16, 0), ([77, 400], 6, 3, 48, 24, 0),
    ([513], 3, 3, 16, 8, 0), ([255, 1030], 8, 2, 256, 32, 0), ([90, 2000], 40, 1, 96, 16, 0), ([1000, 17], 4, 1, 112, 40, 0),
    ([3000], 8, 2, 64, 16, 0), ([900, 40, 5], 8, 2, 64, 16, 1), ([900, 40, 5], 8, 2, 64, 16, 33), ([2000, 700], 8, 8, 128, 16, 512),
    ([5000, 3, 800], 6, 2, 64, 128, 1000), ([50] * 70, 4, 2, 64, 16, 0), ([9000, 20, 4000], 8, 4, 64, 16, 0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,H,G,hd,page,window", DECODE)
def test_decode(lens, H, G, hd, page, window, dtype):
    from vllm_oxide_b200 import kernels
    cache, tables, keys, vals = paged(lens, G, hd, page, sum(lens) + hd)
    S, idle = len(lens), 2
    q = torch.randn(S + idle, H * hd, generator=gen(1)).to(dtype)
    wide = torch.full((S + idle, H * hd + 8), 9.0, dtype=dtype, device=DEV)         # rows that are no tensor of their own
    out = wide[:, :H * hd]
    pos = torch.tensor([n - 1 for n in lens] + [-1] * idle, dtype=torch.int32, device=DEV)
    tab = torch.cat((tables, torch.full((idle, tables.shape[1]), 2 ** 30, dtype=torch.int32, device=DEV)))
    scratch = kernels.kv4_scratch(S + idle, H, G, hd, DEV)
    for _ in range(2):                                       # the scratch is ready for the next launch
        kernels.attn_decode_kv4(q.to(DEV), out, cache, tab, pos, H, G, hd, hd ** -0.5, window=window, scratch=scratch)
    got = out.cpu().double()
    assert (wide[:, H * hd:] == 9).all() and (got[S:] == 0).all() and int(scratch.arrived.abs().sum()) == 0
    for s, n in enumerate(lens):
        ref, size, mag = plain.attend(q[s:s + 1].view(1, H, hd), keys[s], vals[s], torch.tensor([n - 1]), hd ** -0.5, window)
        err = (got[s].view(1, H, hd) - ref).abs()
        tol = tolerance(ref, size, mag, None, dtype)
        assert (err <= tol).all(), (s, n, float((err / tol).max()))


PORTIONS = [  # (context, new) of every request, heads, kv heads, head size, page, window
    ([(0, 1)], 4, 2, 64, 16, 0), ([(0, 5)], 4, 4, 64, 8, 0), ([(0, 64), (64, 64)], 8, 2, 64, 16, 0), ([(0, 130)], 8, 2, 128, 16, 0),
    ([(37, 150), (0, 3), (500, 1)], 6, 2, 128, 16, 0), ([(100, 300)], 8, 2, 64, 64, 0), ([(3, 77), (250, 33)], 6, 3, 48, 24, 0),
    ([(0, 257)], 16, 1, 64, 16, 0), ([(70, 65)], 20, 1, 80, 16, 0), ([(40, 200)], 8, 8, 96, 32, 0), ([(9, 100)], 4, 2, 256, 8, 0),
    ([(0, 300), (700, 200)], 8, 2, 64, 16, 100), ([(1000, 129)], 6, 2, 128, 16, 65), ([(500, 70), (0, 40)], 8, 2, 64, 16, 1),
    ([(1500, 513)], 4, 1, 128, 128, 0), ([(0, 0), (10, 20), (5, 0)], 4, 2, 64, 16, 0), ([(33, 90)], 3, 3, 16, 8, 40),
    ([(2000, 40), (90, 600)], 24, 8, 128, 16, 0), ([(300, 100)], 5, 5, 64, 40, 0), ([(200, 400)], 7, 1, 64, 16, 0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("reqs,H,G,hd,page,window", PORTIONS)
def test_portions(reqs, H, G, hd, page, window, dtype):
    from vllm_oxide_b200 import kernels
    lens = [c + n for c, n in reqs]
    cache, tables, keys, vals = paged(lens, G, hd, page, sum(lens) + hd)
    starts = [0]
    for _, n in reqs:
        starts.append(starts[-1] + n)
    T, behind = starts[-1], 3
    q = torch.randn(T + behind, H * hd, generator=gen(2)).to(dtype)
    wide = torch.full((T + behind, H * hd + 8), 9.0, dtype=dtype, device=DEV)
    out = wide[:, :H * hd]
    kernels.attn_prefill_kv4(q.to(DEV), out, cache, tables, torch.tensor(starts, dtype=torch.int32, device=DEV),
                             torch.tensor([c for c, _ in reqs], dtype=torch.int32, device=DEV), len(reqs), max(n for _, n in reqs), H, G, hd,
                             hd ** -0.5, window=window)
    got = wide.cpu().double()
    assert (got[:, H * hd:] == 9).all() and (got[T:] == 9).all()                    # rows behind the last request stay
    for s, (c, n) in enumerate(reqs):
        if n == 0:
            continue
        rows = slice(starts[s], starts[s] + n)
        ref, size, mag = plain.attend(q[rows].view(n, H, hd), keys[s], vals[s], torch.arange(c, c + n), hd ** -0.5, window)
        err = (got[rows, :H * hd].view(n, H, hd) - ref).abs()
        tol = tolerance(ref, size, mag, None, dtype)
        assert (err <= tol).all(), (s, c, n, float((err / tol).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 48])
def test_a_token_kept_as_nan_reaches_the_rows_that_see_it_and_no_other(hd, dtype):
    from vllm_oxide_b200 import kernels
    H, G, page, n, bad = 4, 2, 16, 150, 100
    g = gen(8)
    k, v = torch.randn(160, G, hd, generator=g), torch.randn(160, G, hd, generator=g)
    v[bad, 0, 3] = math.inf                                  # kv head 0 only: heads 0 and 1
    k[140, 1, 0] = math.nan                                  # kv head 1: heads 2 and 3 from position 140 on
    cache, kk, vv = plain.pack(k, v, page)
    cache = cache.to(DEV)
    tables = torch.arange(10, dtype=torch.int32, device=DEV).view(1, 10)
    q = torch.randn(n, H * hd, generator=g).to(dtype)
    out = torch.empty(n, H * hd, dtype=dtype, device=DEV)
    kernels.attn_prefill_kv4(q.to(DEV), out, cache, tables, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                             torch.zeros(1, dtype=torch.int32, device=DEV), 1, n, H, G, hd, hd ** -0.5)
    got = out.cpu().double().view(n, H, hd)
    assert got[bad:, :2].isnan().all() and not got[:bad, :2].isnan().any()
    assert got[140:, 2:].isnan().all() and not got[:140, 2:].isnan().any()
    ref, size, mag = plain.attend(q[:bad].view(bad, H, hd), kk[:bad], vv[:bad], torch.arange(bad), hd ** -0.5)
    assert ((got[:bad] - ref).abs() <= tolerance(ref, size, mag, None, dtype)).all()
    scratch = kernels.kv4_scratch(4, H, G, hd, DEV)
    pos = torch.tensor([99, 100, 139, 149], dtype=torch.int32, device=DEV)
    o = torch.empty(4, H * hd, dtype=dtype, device=DEV)
    kernels.attn_decode_kv4(q[:4].to(DEV), o, cache, tables.expand(4, 10).contiguous(), pos, H, G, hd, hd ** -0.5, scratch=scratch)
    o = o.cpu().view(4, H, hd)
    assert o[1:, :2].isnan().all() and not o[0].isnan().any() and not o[:3, 2:].isnan().any() and o[3, 2:].isnan().all()
    # in a window that has left it behind, it is not seen
    kernels.attn_decode_kv4(q[:4].to(DEV), (w := torch.empty(4, H * hd, dtype=dtype, device=DEV)), cache, tables.expand(4, 10).contiguous(),
                            pos, H, G, hd, hd ** -0.5, window=39, scratch=scratch)
    w = w.cpu().view(4, H, hd)
    assert not w[0].isnan().any() and w[1, :2].isnan().all() and not w[2, 2:].isnan().any() and not w[2:, :2].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page_no", [-1, 2 ** 30, 12])
def test_a_page_outside_the_pool_makes_its_rows_nan(page_no, dtype):
    """Bounds of the kernels' own: nothing outside the cache is read."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page = 4, 2, 64, 16
    cache, _, _ = plain.pack(torch.randn(192, G, hd, generator=gen(1)), torch.randn(192, G, hd, generator=gen(2)), page)   # 12 pages
    cache = cache.to(DEV)
    tables = torch.arange(12, dtype=torch.int32, device=DEV).repeat(3, 1)
    tables[1, 5] = page_no
    q = torch.randn(3, H * hd, generator=gen(3)).to(dtype).to(DEV)
    out = torch.zeros_like(q)
    scratch = kernels.kv4_scratch(3, H, G, hd, DEV)
    # request 2 claims more tokens than its row of the table has pages
    pos = torch.tensor([191, 100, 192], dtype=torch.int32, device=DEV)
    kernels.attn_decode_kv4(q, out, cache, tables, pos, H, G, hd, hd ** -0.5, scratch=scratch)
    assert not out[0].isnan().any() and out[1].isnan().all() and out[2].isnan().all()
    n = 120
    q = torch.randn(n, H * hd, generator=gen(3)).to(dtype).to(DEV)
    out = torch.zeros_like(q)
    kernels.attn_prefill_kv4(q, out, cache, tables[1:2].contiguous(), torch.tensor([0, n], dtype=torch.int32, device=DEV),
                             torch.zeros(1, dtype=torch.int32, device=DEV), 1, n, H, G, hd, hd ** -0.5)
    assert not out[:80].isnan().any() and out[80:].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("reqs,H,G,hd,page,window", [
    # few rows behind long contexts: blocks share the keys, two, four or eight of them, some with none or with one of the two row tiles only
    ([(5000, 3)], 8, 2, 64, 16, 0), ([(2100, 1)], 4, 4, 128, 16, 0), ([(3000, 90)], 24, 8, 128, 16, 0), ([(2500, 300)], 8, 2, 128, 16, 0),
    ([(4096, 16), (3, 2)], 8, 2, 64, 16, 0), ([(0, 7), (6000, 9), (70, 0), (1025, 5)], 6, 2, 128, 8, 0), ([(5000, 200)], 8, 1, 64, 16, 1500),
    ([(2000, 128)], 2, 2, 64, 24, 600), ([(1100, 260)], 4, 4, 128, 16, 700), ([(3000, 40)], 4, 2, 256, 16, 0), ([(1024, 64)], 20, 1, 80, 16, 0)])
def test_few_rows_behind_long_contexts(reqs, H, G, hd, page, window, dtype):
    test_portions(reqs, H, G, hd, page, window, dtype)


@pytest.mark.parametrize("at", [0, 700, 2047, 4000, 4095])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_nan_token_in_one_blocks_share_of_the_keys(at, dtype):
    from vllm_oxide_b200 import kernels
    H, G, hd, page, L, n = 8, 4, 64, 16, 4096, 6
    g = gen(4)
    k, v = torch.randn(L, G, hd, generator=g), torch.randn(L, G, hd, generator=g)
    v[at, 2, 5] = -math.inf                                  # kv head 2: heads 4 and 5
    cache, kk, vv = plain.pack(k, v, page)
    tables = torch.arange(L // page, dtype=torch.int32, device=DEV).view(1, -1)
    q = torch.randn(n, H * hd, generator=g).to(dtype)
    out = torch.empty(n, H * hd, dtype=dtype, device=DEV)
    kernels.attn_prefill_kv4(q.to(DEV), out, cache.to(DEV), tables, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                             torch.tensor([L - n], dtype=torch.int32, device=DEV), 1, n, H, G, hd, hd ** -0.5)
    got = out.cpu().double().view(n, H, hd)
    sees = torch.arange(L - n, L) >= at
    assert got[sees][:, 4:6].isnan().all() and not got[~sees].isnan().any()
    rest = torch.tensor([0, 1, 2, 3, 6, 7])
    ref, size, mag = plain.attend(q.view(n, H, hd), kk, vv.nan_to_num(), torch.arange(L - n, L), hd ** -0.5)
    assert ((got - ref).abs() <= tolerance(ref, size, mag, None, dtype))[:, rest].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd,n", [(64, 200), (128, 300), (96, 20)])
def test_ranges_far_apart(hd, n, dtype):
    """Runs of 32 keys whose sizes differ by powers of two up to 2^50, zeros among them, queries of all sizes."""
    from vllm_oxide_b200 import kernels
    H, G, page, L = 4, 2, 32, 960
    g = gen(hd + n)
    k, v, q = torch.randn(L, G, hd, generator=g), torch.randn(L, G, hd, generator=g), torch.randn(n, H, hd, generator=g)
    runs = torch.arange(L) // 32
    # keys small where queries are large, so that scores stay in the range where a softmax has more than one key
    q[::3] *= 2.0 ** 30
    q[1::3] *= 2.0 ** -30
    q[5::7] = 0
    k *= (2.0 ** torch.randint(-34, 1, (30,), generator=g).float())[runs, None, None]
    k[::3] *= 2.0 ** -30
    v *= (2.0 ** torch.randint(-25, 26, (30,), generator=g).float())[runs, None, None]
    k[64:128], v[96:160], v[8] = 0, 0, 0
    k, v = (x.to(BF16).float() for x in (k, v))
    cache, kk, vv = plain.pack(k, v, page)
    tables = torch.arange(L // page, dtype=torch.int32, device=DEV).view(1, -1)
    q = q.reshape(n, H * hd).to(dtype)
    out = torch.empty(n, H * hd, dtype=dtype, device=DEV)
    kernels.attn_prefill_kv4(q.to(DEV), out, cache.to(DEV), tables, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                             torch.tensor([L - n], dtype=torch.int32, device=DEV), 1, n, H, G, hd, hd ** -0.5)
    ref, size, mag = plain.attend(q.view(n, H, hd), kk, vv, torch.arange(L - n, L), hd ** -0.5)
    # With scores off by e at most, a weight is by a factor of exp(2 e) at most, and what a row gives by (exp(2 e) - 1) mag; e is 2^-8 of the scores' terms
    # (32 bits: 2^-17). Whatever the weights are they add up to 1, so that it is never off by more than twice the largest value that it sees (2^-7 for roundings).
    off = 2 * (2.0 ** -8 if dtype == BF16 else 2.0 ** -17) * size
    most = torch.stack([vv[:p + 1].abs().amax(0) for p in range(L - n, L)]).repeat_interleave(H // G, 1)
    tol = tolerance(ref, 0.0 * size, mag, None, dtype) + torch.where(off < 40, mag * torch.expm1(off.clamp(max=40)), math.inf).minimum(2 * (1 + 2.0 ** -7) * most)
    assert ((out.cpu().double().view(n, H, hd) - ref).abs() <= tol).all()
    one = torch.empty(n, H * hd, dtype=dtype, device=DEV)
    scratch = kernels.kv4_scratch(n, H, G, hd, DEV)
    kernels.attn_decode_kv4(q.to(DEV), one, cache.to(DEV), tables.expand(n, -1).contiguous(), torch.arange(L - n, L, dtype=torch.int32, device=DEV),
                            H, G, hd, hd ** -0.5, scratch=scratch)
    assert ((one.cpu().double().view(n, H, hd) - ref).abs() <= tol).all()


@pytest.mark.parametrize("what", ["portions", "few rows", "single tokens"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_call_gives_the_same_bits(what, dtype):
    from vllm_oxide_b200 import kernels
    H, G, hd, page = 24, 8, 128, 16
    lens = [2600, 40, 3000] if what != "portions" else [700, 40, 900]
    cache, tables, _, _ = paged(lens, G, hd, page, 5)
    new = {"portions": [500, 40, 300], "few rows": [5, 1, 3], "single tokens": [1, 1, 1]}[what]
    starts = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([a - b for a, b in zip(lens, new)], dtype=torch.int32, device=DEV)
    q = torch.randn(sum(new), H * hd, generator=gen(6)).to(dtype).to(DEV)
    scratch = kernels.kv4_scratch(3, H, G, hd, DEV)
    first = None
    for _ in range(20):
        out = torch.full_like(q, 5.0)
        if what == "single tokens":
            kernels.attn_decode_kv4(q, out, cache, tables, ctx, H, G, hd, hd ** -0.5, scratch=scratch)
        else:
            kernels.attn_prefill_kv4(q, out, cache, tables, starts, ctx, 3, max(new), H, G, hd, hd ** -0.5)
        first = out if first is None else first
        assert torch.equal(out, first)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_captured_step_follows_its_inputs(dtype):
    """append, attention of single tokens and of portions in one graph, replayed at other positions, slots and lengths."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page, S, n = 8, 2, 64, 16, 3, 20
    cache, tables, _, _ = paged([2500] * S, G, hd, page, 11)
    f = freq(hd).to(DEV)
    x = torch.randn(S + n, (H + 2 * G) * hd, generator=gen(12)).to(dtype).to(DEV)
    ints = torch.zeros(4, S + n, dtype=torch.int32, device=DEV)
    positions, slots, starts, contexts = ints
    scratch = kernels.kv4_scratch(S, H, G, hd, DEV)
    out = torch.empty(S + n, H * hd, dtype=dtype, device=DEV)
    q_out = torch.empty_like(out)

    def step():
        kernels.kv4_append(x[:, :H * hd], x[:, H * hd:(H + G) * hd], x[:, (H + G) * hd:], positions, slots, f, cache, H, G, hd, q_out=q_out)
        kernels.attn_decode_kv4(q_out[:S], out[:S], cache, tables, positions, H, G, hd, hd ** -0.5, scratch=scratch)
        kernels.attn_prefill_kv4(q_out, out, cache, tables[1:2], starts, contexts, 1, n, H, G, hd, hd ** -0.5)

    def place(lens, context):
        pos = torch.tensor([m - 1 for m in lens] + list(range(context, context + n)), dtype=torch.int32)
        rows = torch.tensor(list(range(S)) + [1] * n)
        positions.copy_(pos)
        slots.copy_(tables.cpu()[rows, pos.long() // page] * page + pos % page)
        starts[:2] = torch.tensor([S, S + n], dtype=torch.int32)
        contexts[:1] = context

    place([5, 900, 40], 300)
    step()
    torch.cuda.synchronize()
    before = cache.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens, context in (([2400, 17, 600], 1900), ([1, 2, 3], 2), ([700, 2100, 2500], 100)):            # (a token of request 1 and its portion never at one position: one slot a token)
        place(lens, context)
        cache.copy_(before)
        graph.replay()
        got, kept = out.clone(), cache.clone()
        cache.copy_(before)
        out.zero_()
        step()
        assert torch.equal(got, out) and torch.equal(kept, cache) and not got[:1].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_streams_at_once(dtype):
    """Each with scratch of its own; the kernels share nothing else."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page = 24, 8, 128, 16
    cache, tables, _, _ = paged([3000, 700], G, hd, page, 21)
    q = torch.randn(40, H * hd, generator=gen(22)).to(dtype).to(DEV)
    pos = torch.tensor([2999, 500], dtype=torch.int32, device=DEV)
    starts, ctx = torch.tensor([0, 30, 40], dtype=torch.int32, device=DEV), torch.tensor([2970, 600], dtype=torch.int32, device=DEV)

    def both(scratch, one, many):
        kernels.attn_decode_kv4(q[:2], one, cache, tables, pos, H, G, hd, hd ** -0.5, scratch=scratch)
        kernels.attn_prefill_kv4(q, many, cache, tables, starts, ctx, 2, 30, H, G, hd, hd ** -0.5)

    want = [torch.empty(2, H * hd, dtype=dtype, device=DEV), torch.empty_like(q)]
    both(kernels.kv4_scratch(2, H, G, hd, DEV), *want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    scratches = [kernels.kv4_scratch(2, H, G, hd, DEV) for _ in streams]
    outs = [[[torch.empty_like(w) for w in want] for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                both(scratches[s], *outs[s][i])
    torch.cuda.synchronize()
    for per_stream in outs:
        for got in per_stream:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_cache_beyond_32_bits_of_bytes(dtype):
    """The same requests at both ends of a pool of 5 GB give the same bits."""
    from vllm_oxide_b200 import kernels
    H, G, hd, page, L, n = 8, 8, 128, 64, 500, 70
    pages = 5 * 2 ** 30 // (G * page * plain.width(hd))
    cache = torch.empty(pages, G, page, plain.width(hd), dtype=torch.uint8, device=DEV)
    g = gen(31)
    qkv = torch.randn(L, (H + 2 * G) * hd, generator=g).to(dtype).to(DEV)
    positions = torch.arange(L, dtype=torch.int32, device=DEV)
    need = -(-L // page)
    got = []
    for first in (0, pages - need):
        table = torch.arange(first, first + need, dtype=torch.int32, device=DEV).view(1, -1)
        slots = first * page + positions
        q = torch.empty(L, H * hd, dtype=dtype, device=DEV)
        kernels.kv4_append(qkv[:, :H * hd], qkv[:, H * hd:(H + G) * hd], qkv[:, (H + G) * hd:], positions, slots, freq(hd).to(DEV), cache, H, G, hd, q_out=q)
        k, v = (torch.empty(L, G * hd, dtype=dtype, device=DEV) for _ in range(2))
        kernels.kv4_read(cache, slots, k, v, G, hd)
        one, many = torch.empty(1, H * hd, dtype=dtype, device=DEV), torch.empty(n, H * hd, dtype=dtype, device=DEV)
        kernels.attn_decode_kv4(q[-1:], one, cache, table, positions[-1:], H, G, hd, hd ** -0.5, scratch=kernels.kv4_scratch(1, H, G, hd, DEV))
        kernels.attn_prefill_kv4(q[-n:], many, cache, table, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                                 torch.tensor([L - n], dtype=torch.int32, device=DEV), 1, n, H, G, hd, hd ** -0.5)
        got.append((q, k, v, one, many))
    for a, b in zip(*got):
        assert torch.equal(a, b) and not a.isnan().any()
    (q, k, v, one, many) = (x.cpu() for x in got[0])
    ref, size, mag = plain.attend(q[-n:].view(n, H, hd), k.double().view(L, G, hd), v.double().view(L, G, hd), torch.arange(L - n, L), hd ** -0.5)
    # (keys and values as read back are rounded to the type: half a step of them more)
    tol = tolerance(ref, size, mag, None, dtype) + HALF[dtype] * (2 * size * (mag + ref.abs()) + mag)
    assert ((many.double().view(n, H, hd) - ref).abs() <= tol).all() and ((one.double().view(1, H, hd) - ref[-1:]).abs() <= tol[-1:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_at_odd_addresses_and_calls_without_rows(hd, dtype):
    from vllm_oxide_b200 import kernels
    H, G, page, lens, new = 8, 2, 16, [2000, 60], [9, 40]
    cache, tables, keys, vals = paged(lens, G, hd, page, hd)
    rows = sum(new)
    wide = torch.randn(rows, H * hd + 3, generator=gen(41)).to(dtype).to(DEV)
    q, out = wide[:, 1:1 + H * hd], torch.full((rows, H * hd + 5), 3.0, dtype=dtype, device=DEV)[:, 3:3 + H * hd]
    starts = torch.tensor([0, new[0], rows], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([a - b for a, b in zip(lens, new)], dtype=torch.int32, device=DEV)
    scratch = kernels.kv4_scratch(2, H, G, hd, DEV)

    def portions(seqs, longest):
        kernels.attn_prefill_kv4(q, out, cache, tables, starts, ctx, seqs, longest, H, G, hd, hd ** -0.5)

    def single(n):
        kernels.attn_decode_kv4(q[:n], out[:n], cache, tables, ctx, H, G, hd, hd ** -0.5, scratch=scratch)

    portions(0, 40)
    portions(2, 0)
    single(0)
    assert (out == 3).all()
    portions(2, 40)
    got, at = out.cpu().double(), 0
    for s, n in enumerate(new):
        ref, size, mag = plain.attend(q.cpu()[at:at + n].reshape(n, H, hd), keys[s], vals[s], torch.arange(lens[s] - n, lens[s]), hd ** -0.5)
        assert ((got[at:at + n].view(n, H, hd) - ref).abs() <= tolerance(ref, size, mag, None, dtype)).all()
        at += n
    single(2)
    got = out.cpu().double()
    for s in range(2):
        n = int(ctx[s]) + 1
        ref, size, mag = plain.attend(q.cpu()[s:s + 1].reshape(1, H, hd), keys[s][:n], vals[s][:n], torch.tensor([n - 1]), hd ** -0.5)
        assert ((got[s].view(1, H, hd) - ref).abs() <= tolerance(ref, size, mag, None, dtype)).all()
