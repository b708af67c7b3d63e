"""Four-bit caches and matrices, and log-probabilities, against the 64-bit
oracle: sizes and masks at the borders of blocks, tiles, partitions and parts,
what the device finds in its own memory, streams and graphs."""
import itertools

import numpy as np
import pytest
import torch

from hexgen2_amd import fp4, logprobs, ops
from oracle import mx_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def randn(shape, seed, dtype, device, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(device)


def wide(t):
    return t.detach().cpu().double().numpy()


def same(got, want):
    """Bit-equal values (NaN with NaN)."""
    return np.array_equal(wide(got), want.astype(wide(got).dtype), equal_nan=True)


def in_dtype(values, dtype):
    """Float64 values as they read after one rounding to ``dtype`` (torch goes
    through float32, exactly for these: two significant bits)."""
    return torch.from_numpy(values).to(dtype).double().numpy()


# ------------------------------------------------------- rows in and out ---


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 96, 2048, 8192 + 32])
def test_quantize_and_back(device, dtype, width):
    x = randn((5, width), width, dtype, device, 3.0)
    x[0, :32] = 0
    x[1, 3] = 40  # one far larger than its block
    w = fp4.quantize(x)
    codes, powers = oracle.quantize(wide(x))
    assert np.array_equal(w.powers.cpu().numpy(), powers)
    assert np.array_equal(w.codes.cpu().numpy(), oracle.pack(codes))
    for to in DTYPES:
        assert same(fp4.dequantize(w, to), in_dtype(oracle.values(codes, powers), to))


@pytest.mark.parametrize("power", [-125, -20, 0, 13, 126])
def test_quantize_halfway_values(device, power):
    x = np.zeros((2, 32))
    x[0, :16] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 3]
    x[1, :8] = np.array([1.5, 0.3, 0.7, -1.2, 0.1, -0.9, 1.1, 0.625]) * 2  # its largest is exactly 3: power - 1
    if power == 126:
        x = np.clip(x, -3.5, 3.5)
    x *= 2.0 ** power
    w = fp4.quantize(torch.from_numpy(x).float().to(device))
    codes, powers = oracle.quantize(x)
    assert np.array_equal(w.codes.cpu().numpy(), oracle.pack(codes)) and np.array_equal(w.powers.cpu().numpy(), powers)


def test_quantize_marks_what_is_not_finite(device):
    x = randn((4, 64), 1, torch.float32, device)
    x[0, 5], x[1, 40], x[2, 63] = float("inf"), float("nan"), -float("inf")
    x[3, :32] = 1e-42  # subnormal
    got = fp4.dequantize(fp4.quantize(x), torch.float32)
    assert same(got, oracle.rounded(wide(x)))
    assert torch.isnan(got[0, :32]).all() and torch.isfinite(got[0, 32:]).all()


def test_every_byte_and_code_dequantizes(device):
    codes = np.tile(np.arange(32) % 16, (256, 1))
    powers = np.arange(256)[:, None]
    w = fp4.Fp4Tensor(torch.from_numpy(oracle.pack(codes)).to(device), torch.from_numpy(powers.astype(np.uint8)).to(device))
    want = oracle.values(codes, powers)
    assert same(fp4.dequantize(w, torch.float32), in_dtype(want, torch.float32))
    assert same(fp4.dequantize(w, torch.bfloat16), in_dtype(want, torch.bfloat16))
    assert same(fp4.dequantize(w, torch.float16), in_dtype(want, torch.float16))


GEOMETRIES = [(8, 128), (1, 128), (4, 64), (3, 32), (2, 256), (32, 128)]


@pytest.mark.parametrize("dtype,geometry", itertools.product(DTYPES, GEOMETRIES))
def test_store_and_load(device, dtype, geometry):
    heads, d = geometry
    kv = randn((2, 5, 2, heads, d), heads * d, dtype, device)
    cache = fp4.kv_cache(3, 9, heads, d, device).fill_(0xAB)
    fp4.store_kv(cache, kv, position_bias=3)
    want = oracle.rows(wide(kv))
    used = 2 * heads * (d // 2 + d // 32)
    assert np.array_equal(cache[:2, 3:8, :used].cpu().numpy(), want[..., :used])
    rest = cache.clone()
    rest[:2, 3:8] = 0xAB
    assert (rest == 0xAB).all()  # nothing else is touched, another sequence included
    assert (cache[:2, 3:8, used:] == 0xAB).all()
    assert same(fp4.load_kv(cache[:2], 5, heads, d, dtype, position_bias=3), in_dtype(oracle.rounded(wide(kv)), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_and_load_of_strided_and_unaligned_rows(device, dtype):
    heads, d = 3, 64
    base = randn((2 * 4 * 2 * heads * d * 2 + 11,), 5, dtype, device)
    for start, strides in ((0, (4 * 800, 800, 400)), (1, (3 * 391 + 4, 391, heads * d)), (3, (400, 800, 2000))):
        kv = base.as_strided((2, 2, 2, heads, d), (*strides, d, 1), start)
        cache = fp4.kv_cache(2, 40, heads, d, device)[:, 3:30]  # rows of a longer cache
        fp4.store_kv(cache, kv, position_bias=24)
        want = oracle.rounded(wide(kv))
        assert same(fp4.load_kv(cache, 2, heads, d, dtype, position_bias=24), in_dtype(want, dtype))
        out = torch.full((2, 2, 2, heads * d + 1), 7.0, dtype=dtype, device=device)
        view = out[..., 1:].unflatten(-1, (heads, d))
        fp4.load_kv(cache, 2, heads, d, dtype, position_bias=24, out=view)
        assert same(view, in_dtype(want, dtype)) and (out[..., 0] == 7).all()


def test_positions_from_the_device(device):
    heads, d = 2, 64
    kv = randn((4, 1, 2, heads, d), 2, torch.bfloat16, device)
    cache = fp4.kv_cache(4, 6, heads, d, device).zero_()
    at = torch.tensor([5, 0, 6, -1], dtype=torch.int32, device=device)
    ops.device_status(device)
    fp4.store_kv(cache, kv, at)
    with pytest.raises(ValueError, match="append position"):
        ops.check_device_status(device)
    want = oracle.rows(wide(kv))[:, 0]
    assert np.array_equal(cache[0, 5].cpu().numpy(), want[0]) and np.array_equal(cache[1, 0].cpu().numpy(), want[1])
    assert not cache[2:].any() and not cache[0, :5].any()
    got = fp4.load_kv(cache, 1, heads, d, torch.bfloat16, at)
    with pytest.raises(ValueError, match="load"):
        ops.check_device_status(device)
    assert same(got[:2], in_dtype(oracle.rounded(wide(kv[:2])), torch.bfloat16)) and not got[2:].any()
    # one position beyond the int32 range when the bias is added
    at.fill_(2 ** 31 - 1)
    fp4.store_kv(cache, kv, at, position_bias=2 ** 31 - 1)
    assert ops.device_status(device) == 1


def test_rows_of_nothing(device):
    cache = fp4.kv_cache(2, 4, 2, 64, device)
    fp4.store_kv(cache, torch.empty(2, 0, 2, 2, 64, device=device))
    assert fp4.load_kv(cache, 0, 2, 64, torch.float16).shape == (2, 0, 2, 2, 64)
    assert fp4.quantize(torch.empty(0, 64, device=device)).codes.shape == (0, 32)
    assert fp4.linear(torch.empty(0, 64, device=device), fp4.quantize(torch.zeros(3, 64, device=device))).shape == (0, 3)


def test_handoff_carries_four_bit_rows(device):
    heads, d, lens = 8, 128, [3, 0, 7]
    layers = [fp4.kv_cache(3, 8, heads, d, device) for _ in range(2)]
    kv = [randn((3, 8, 2, heads, d), i, torch.bfloat16, device) for i in range(2)]
    for cache, x in zip(layers, kv):
        fp4.store_kv(cache, x)
    packed = ops.pack_live(layers, lens)
    decode = [torch.zeros_like(layers[0]) for _ in range(2)]
    ops.unpack_live(packed, decode, lens)
    for cache, x in zip(decode, kv):
        got = wide(fp4.load_kv(cache, 8, heads, d, torch.bfloat16))
        want = oracle.rounded(wide(x))
        for b, n in enumerate(lens):
            assert np.array_equal(got[b, :n], want[b, :n]) and not got[b, n:].any()


# -------------------------------------------------------------- attention ---


def attend_tolerance(q, kv, want, dtype):
    """Half a step of the type; and in units of the largest value: twice the
    relative error of a probability -- its score's (sums of d products in
    fp32, a few steps of the score itself), its rounding to two 8-bit
    terms (three for fp32) -- and the fp32 sums over the keys."""
    d, n = q.shape[-1], kv.shape[1]
    size = np.abs(q).sum(-1).max() * np.abs(kv[:, :, 0]).max() * d ** -0.5  # at least any sum |q k| scale
    p = 2.0 ** -16 if dtype != torch.float32 else 2.0 ** -23
    relative = 2 * (d * 2.0 ** -24 * min(size, 64.0) + 2.0 ** -19 + p) + n * 2.0 ** -24
    return torch.finfo(dtype).eps / 2 * np.abs(want) + relative * np.abs(kv[:, :, 1]).max() + 1e-30


def make_cache(kv, capacity, device, stale=0xFF):
    """A 4-bit cache of ``kv [B, S, 2, H, D]``; rows behind hold bytes that
    read as NaN."""
    b, s, _, h, d = kv.shape
    cache = fp4.kv_cache(b, capacity, h, d, device).fill_(stale)
    fp4.store_kv(cache, kv)
    return cache


CASES = [
    # q_heads, kv_heads, head_dim, lens, q_len, partition
    (8, 8, 128, [1, 33, 64], 1, 0), (32, 8, 128, [0, 31, 200], 1, 64), (8, 1, 128, [97, 5], 1, 32),
    (32, 4, 64, [577], 1, 0), (32, 1, 64, [65, 1], 1, 32), (4, 2, 32, [40, 0, 1], 1, 0), (6, 2, 256, [70, 129], 1, 64),
    (40, 2, 128, [33], 1, 0), (8, 2, 128, [40, 64], 3, 32), (4, 4, 64, [90, 7], 9, 64), (2, 1, 32, [35], 20, 0),
    (8, 2, 256, [3, 50], 4, 32), (8, 2, 128, [150, 61], 40, 0), (4, 1, 64, [130, 200], 70, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case,causal", [(i, causal) for i in range(len(CASES)) for causal in (False, True)
                                         if not causal or CASES[i][4] > 1])
def test_attention(device, dtype, case, causal):
    hq, h, d, lens, t, partition = CASES[case]
    kv = randn((len(lens), max(lens), 2, h, d), case, dtype, device)
    q = randn((len(lens), t, hq, d), 100 + case, dtype, device, 2.0)
    cache = make_cache(kv, max(lens) + 5, device)
    seqlens = torch.tensor(lens, dtype=torch.int32, device=device)
    for b, n in enumerate(lens):
        cache[b, n:] = 0xFF  # NaN behind every sequence's own length
    out = torch.full_like(q, 9.0)
    got = fp4.decode_attention(q, cache, h, max_seqlen=max(lens), seqlens=seqlens, causal=causal, out=out,
                               partition=partition)
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, lens, causal)
    assert got is out
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()
    for b, n in enumerate(lens):  # rows without keys are zero, not merely small
        none = max(0, t - n) if causal else (t if n == 0 else 0)
        assert not got[b, :none].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,hq,h,d,longest,q_len,partition", [
    (2, 4, 2, 64, 700, 1, 32),     # 22 partitions: eight waves join a row
    (9, 2, 1, 32, 260, 2, 128),    # joined by one wave; a sequence of one key beside them
    (70, 8, 4, 64, 300, 1, 0),     # more workgroups than CUs: four waves each
    (1, 2, 1, 128, 1100, 1, 0),    # split by the rule
    (3, 24, 1, 32, 90, 6, 0),      # fewer (sequence, partition) pairs than XCDs, more with the row tiles
    (257, 1, 1, 32, 40, 1, 0),
])
def test_attention_of_many_workgroups(device, dtype, batch, hq, h, d, longest, q_len, partition):
    lens = [1 + (i * 977 + longest - 1) % longest for i in range(batch)]  # the first one longest
    kv = randn((batch, longest, 2, h, d), batch, dtype, device)
    q = randn((batch, q_len, hq, d), 9, dtype, device, 2.0)
    cache = make_cache(kv, longest, device)
    for b, n in enumerate(lens):
        cache[b, n:] = 0xFF
    got = fp4.decode_attention(q, cache, h, max_seqlen=longest, causal=True, partition=partition,
                               seqlens=torch.tensor(lens, dtype=torch.int32, device=device))
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, lens, q_len > 1)
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("geometry", [(32, 8, 128), (8, 1, 128), (32, 4, 64), (4, 2, 32), (4, 2, 256), (40, 2, 64)])
@pytest.mark.parametrize("partition", [0, 32])
def test_fused_append(device, dtype, geometry, partition):
    hq, h, d = geometry
    lens = [0, 31, 32, 63, 100]  # the new row alone, and at either side of a tile
    kv = randn((5, 101, 2, h, d), 3, dtype, device)
    new = randn((5, 1, 2, h, d), 4, dtype, device, 2.0)
    q = randn((5, 1, hq, d), 5, dtype, device, 2.0)
    cache = make_cache(kv, 101, device)
    before = cache.clone()
    seqlens = torch.tensor(lens, dtype=torch.int32, device=device)
    got = fp4.decode_attention(q, cache, h, max_seqlen=101, seqlens=seqlens, kv_new=new, partition=partition)
    stored = oracle.rounded(wide(kv))
    for b, n in enumerate(lens):
        stored[b, n] = oracle.rounded(wide(new[b, 0]))
    want = oracle.attend(wide(q), stored, [n + 1 for n in lens])
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()
    appended = before.clone()
    fp4.store_kv(appended, new, seqlens)
    used = 2 * h * (d // 2 + d // 32)
    assert torch.equal(cache[..., :used], appended[..., :used])  # that row, as store_kv writes it, and no other
    # attending afterwards gives the very same bits
    again = fp4.decode_attention(q, cache, h, max_seqlen=101, seqlens=seqlens, seqlen_bias=1, partition=partition)
    assert torch.equal(got, again)


def test_lengths_from_the_device_are_clamped(device):
    kv = randn((3, 40, 2, 2, 64), 3, torch.float16, device)
    q = randn((3, 1, 4, 64), 5, torch.float16, device)
    cache = make_cache(kv, 40, device)
    before = cache.clone()
    ops.device_status(device)
    lens = torch.tensor([50, -7, 12], dtype=torch.int32, device=device)
    new = randn((3, 1, 2, 2, 64), 6, torch.float16, device)
    got = fp4.decode_attention(q, cache, 2, max_seqlen=30, seqlens=lens, kv_new=new)
    assert ops.device_status(device) == 2
    stored = oracle.rounded(wide(kv))
    stored[2, 12] = oracle.rounded(wide(new[2, 0]))
    want = oracle.attend(wide(q), stored, [30, 0, 13])
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, torch.float16)).all()
    assert torch.equal(cache[:2], before[:2]) and not torch.equal(cache[2, 12], before[2, 12])


@pytest.mark.parametrize("q_len", [1, 3, 40])
def test_nan_reaches_the_rows_that_attend_it(device, q_len):
    lens = [70, 64]
    kv = randn((2, 70, 2, 2, 64), 7, torch.bfloat16, device)
    kv[0, 68, 0, 1, 3] = float("nan")   # a key: every output of head 1 that attends it
    kv[0, 69, 1, 0, 40] = float("inf")  # a value: the second block of head 0's outputs
    q = randn((2, q_len, 4, 64), 8, torch.bfloat16, device)
    cache = make_cache(kv, 80, device)
    got = wide(fp4.decode_attention(q, cache, 2, max_seqlen=70, seqlens=torch.tensor(lens, dtype=torch.int32, device=device),
                                    causal=True))
    nan = np.isnan(got)
    for t in range(q_len):
        n = 70 - (q_len - 1 - t)
        assert nan[0, t, 2:].all() == (n > 68) and nan[0, t, 2:].any() == (n > 68)
        assert nan[0, t, :2, 32:].all() == (n > 69) and nan[0, t, :2, 32:].any() == (n > 69) and not nan[0, t, :2, :32].any()
    assert not nan[1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_len", [3, 20, 200])
@pytest.mark.parametrize("d", [32, 64, 256])
def test_values_past_the_largest_float_reach_the_rows_that_attend_them(device, dtype, q_len, d):
    """A value rounded to 2^128, and such codes of the two largest powers."""
    kv = randn((1, 70, 2, 2, d), 7, dtype, device)
    kv[0, 69, 1, 0, d - 3] = 3.3e38
    q = torch.zeros((1, q_len, 4, d), dtype=dtype, device=device)  # every key counts alike
    cache = make_cache(kv, 70, device)
    power = 2 * d + 2 * (d // 32)  # the first of the values' powers, behind 2 d bytes of elements and the keys' powers
    assert cache[0, 69, power + d // 32 - 1] == 253
    for byte, code, finite in ((253, None, False), (254, 4, False), (254, 0xC, False), (254, 3, True), (253, 5, True), (253, 0xF, False)):
        cache[0, 69, power + d // 32 - 1] = byte
        if code is not None:
            start = d + d // 2 - 16  # head 0's last block of values
            cache[0, 69, start:start + 16] = 0
            cache[0, 69, start + 14] = code << 4
        got = wide(fp4.decode_attention(q, cache, 2, max_seqlen=70, seqlen_bias=70, causal=True))
        assert np.isfinite(got[0, :-1]).all() and np.isfinite(got[0, -1, 2:]).all() and np.isfinite(got[0, -1, :2, :d - 32]).all()
        assert np.isfinite(got[0, -1, :2, d - 3]).all() == finite, (byte, code)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("partition", [0, 32])
@pytest.mark.parametrize("q_len", [1, 9])
def test_scores_far_below_zero(device, dtype, partition, q_len):
    """Equal scores of -2^114 and below: the mean of the values."""
    kv = randn((1, 70, 2, 1, 64), 3, dtype, device)
    kv[:, :, 0] = -2.0 ** 60
    q = torch.full((1, q_len, 2, 64), 2.0 ** 50, dtype=dtype, device=device)
    got = fp4.decode_attention(q, make_cache(kv, 70, device), 1, max_seqlen=70, seqlen_bias=70, partition=partition)
    values = oracle.rounded(wide(kv))[0, :, 1, 0]
    tol = torch.finfo(dtype).eps / 2 * np.abs(values.mean(0)) + 70 * 2.0 ** -24 * np.abs(values).max() + 2.0 ** -16 * np.abs(values).max()
    assert (np.abs(wide(got) - values.mean(0)) <= tol).all()


def test_an_infinite_query(device):
    kv = randn((1, 9, 2, 1, 64), 7, torch.float16, device)
    q = randn((1, 1, 2, 64), 8, torch.float16, device)
    q[0, 0, 0, 1] = float("inf")
    got = fp4.decode_attention(q, make_cache(kv, 9, device), 1, max_seqlen=9, seqlen_bias=9)
    assert torch.isnan(got[0, 0, 0]).all() and torch.isfinite(got[0, 0, 1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_over_far_powers(device, dtype):
    """Powers beyond fp16's range on either side, products within fp32's."""
    kv = randn((1, 70, 2, 2, 64), 3, dtype, device)
    kv[:, :, 0] *= 2.0 ** -60
    kv[:, :35, 1] *= 2.0 ** 50
    kv[:, 35:, 1] *= 2.0 ** -80
    q = (randn((1, 1, 4, 64), 5, dtype, device) * 2.0 ** 60).to(dtype)
    got = fp4.decode_attention(q, make_cache(kv, 70, device), 2, max_seqlen=70, seqlen_bias=70)
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, [70])
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()


def test_attention_of_strided_rows(device):
    heads, d = 2, 64
    wide_q = randn((2, 3, 5 * heads * d + 1), 1, torch.bfloat16, device)
    q = wide_q[..., 1:1 + 4 * d].unflatten(-1, (4, d))  # rows at odd addresses, as a slice of a joined product
    kv = randn((2, 40, 2, heads, d), 2, torch.bfloat16, device)
    cache = fp4.kv_cache(2, 90, heads, d, device).fill_(0xFF)[:, 20:70]
    fp4.store_kv(cache, kv)
    out = torch.zeros((2, 3, 4 * d + 3), dtype=torch.bfloat16, device=device)
    view = out[..., 3:].unflatten(-1, (4, d))
    fp4.decode_attention(q, cache, heads, max_seqlen=40, seqlen_bias=40, causal=True, out=view)
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, [40, 40], True)
    assert (np.abs(wide(view) - want) <= attend_tolerance(wide(q), stored, want, torch.bfloat16)).all()
    assert not out[..., :3].any()


def test_attention_of_padded_rows_after_a_single_position(device):
    """Two views of a cache whose rows lie further apart than they are long, the
    first of one position (whose stride says nothing)."""
    kv = randn((1, 8, 2, 2, 64), 1, torch.float16, device)
    q = randn((1, 1, 4, 64), 2, torch.float16, device)
    packed = make_cache(kv, 8, device)
    padded = torch.full((1, 8, 192), 0xFF, dtype=torch.uint8, device=device)[..., :144]
    padded.copy_(packed)
    for n in (1, 8, 5):
        got = fp4.decode_attention(q, padded[:, :n], 2, max_seqlen=n, seqlen_bias=n)
        assert torch.equal(got, fp4.decode_attention(q, packed[:, :n], 2, max_seqlen=n, seqlen_bias=n)), n


@pytest.mark.parametrize("q_len,partition", [(1, 0), (1, 32), (5, 0), (5, 64), (130, 0)])
def test_attention_in_place(device, q_len, partition):
    kv = randn((2, 200, 2, 2, 64), 1, torch.bfloat16, device)
    q = randn((2, q_len, 8, 64), 2, torch.bfloat16, device)
    cache = make_cache(kv, 200, device)
    want = fp4.decode_attention(q, cache, 2, max_seqlen=200, seqlen_bias=200, causal=True, partition=partition)
    assert fp4.decode_attention(q, cache, 2, max_seqlen=200, seqlen_bias=200, causal=True, partition=partition, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("partition", [0, 32])
def test_the_rounding_of_probabilities(device, dtype, partition):
    """Two keys of one step whose values cancel but for the difference of their probabilities,
    1 and exp(-gap): both terms of the second, below 1, are rounded, 2^-9 and then 2^-18 off at
    most; half of that times the value 6 is left in the output, beside
    fp32's errors (2^-22 for the exponential, the sum and the quotient) and the
    output's own rounding."""
    d, rows = 64, 32
    kv = np.zeros((1, 64, 2, 1, d))
    kv[0, 0, 0, 0, 0] = 1
    kv[0, 1:, 0, 0, 2], kv[0, 20, 0, 0, 2] = 6, 0  # the others score -600
    kv[0, 0, 1], kv[0, 20, 1] = 6, -6
    q = torch.zeros((1, 1, rows, d), dtype=dtype, device=device)
    q[0, 0, :, 0] = torch.from_numpy(np.random.default_rng(1).uniform(2.0 ** -14, 2.0 ** -13, rows)).to(dtype).to(device)
    q[0, 0, :, 2] = -100
    cache = make_cache(torch.from_numpy(kv).to(dtype).to(device), 64, device)
    got = fp4.decode_attention(q, cache, 1, max_seqlen=64, seqlen_bias=64, softmax_scale=1.0, partition=partition)
    want = oracle.attend(wide(q), oracle.rounded(kv), [64], scale=1.0)
    assert (np.abs(wide(got) - want) <= torch.finfo(dtype).eps / 2 * np.abs(want) + 6 * (2.0 ** -19 + 2.0 ** -22)).all()


def takes_out(q, cache, kv_heads, longest, causal):
    """Whether this call attends a copy of the cache in 16 bits: its workspace is
    another than the same call's at an odd address, which reads four bits."""
    b, t, hq, d = q.shape
    odd = torch.empty((b, t, hq * d + 1), dtype=q.dtype, device=q.device)[..., 1:].unflatten(-1, (hq, d))
    return (fp4.attend_workspace_bytes(q, cache, kv_heads, longest, causal=causal)
            != fp4.attend_workspace_bytes(odd, cache, kv_heads, longest, causal=causal))


CHUNKS = [
    # q_heads, kv_heads, head_dim, lens, q_len: 25 and more tiles of 16 rows per KV head
    (4, 1, 128, [130, 0, 257], 100), (8, 2, 64, [300, 97], 128), (2, 1, 64, [90], 200), (4, 1, 128, [2900], 110),
    (8, 1, 64, [701, 40], 70),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case,causal", itertools.product(range(len(CHUNKS)), (False, True)))
def test_attention_of_a_chunk(device, dtype, case, causal):
    hq, h, d, lens, t = CHUNKS[case]
    b = len(lens)
    kv = randn((b, max(lens), 2, h, d), case, dtype, device)
    q = randn((b, t, hq, d), 100 + case, dtype, device, 2.0)
    cache = make_cache(kv, max(lens) + 5, device)
    for i, n in enumerate(lens):
        cache[i, n:] = 0xFF  # NaN behind every sequence's own length
    seqlens = torch.tensor(lens, dtype=torch.int32, device=device)
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, lens, causal)
    tol = attend_tolerance(wide(q), stored, want, dtype)
    rows = torch.zeros((b, t, hq * d + 3), dtype=dtype, device=device)
    odd_out = rows[..., 3:].unflatten(-1, (hq, d))
    odd_q = torch.zeros((b, t, hq * d + 1), dtype=dtype, device=device)[..., 1:].unflatten(-1, (hq, d)).copy_(q)
    for query, out in ((q, None), (q, odd_out), (odd_q, None), (odd_q, odd_out)):
        assert takes_out(query, cache, h, max(lens), causal) == (dtype == torch.bfloat16 and query is q)
        got = fp4.decode_attention(query, cache, h, max_seqlen=max(lens), seqlens=seqlens, causal=causal, out=out)
        assert (np.abs(wide(got) - want) <= tol).all()
        for i, n in enumerate(lens):
            assert not got[i, :max(0, t - n) if causal else (t if n == 0 else 0)].any()
    assert not rows[..., :3].any()


def test_nan_reaches_the_rows_of_a_chunk_that_attend_it(device):
    cache = fp4.kv_cache(2, 80, 2, 64, device)
    assert takes_out(torch.empty((2, 200, 4, 64), dtype=torch.bfloat16, device=device), cache, 2, 70, True)
    test_nan_reaches_the_rows_that_attend_it(device, 200)


@pytest.mark.parametrize("source", [torch.float16, torch.float32])
@pytest.mark.parametrize("q_len", [40, 130])
def test_chunks_over_values_that_fp16_does_not_hold(device, source, q_len):
    """fp16 queries on either side of the tiles that bf16 ones are taken out at:
    fp16 values from 57344 up, stored as 65536; keys of powers far from fp16's."""
    kv = randn((2, 150, 2, 2, 64), 3, torch.float32, device)
    kv[:, :, 1, :, :32] *= 2.0 ** 13
    kv[0, ::7, 1, 0, 5], kv[0, 1::7, 1, 0, 5] = 60000, -60000  # their means stay within fp16
    kv[:, :, 1].clamp_(-60000, 60000)
    kv[:, :, 0, 1] *= 2.0 ** (14 if source == torch.float16 else 20)
    if source == torch.float16:
        kv[:, :, 0].clamp_(-65000, 65000)
    kv = kv.to(source)
    q = randn((2, q_len, 8, 64), 4, torch.float16, device, 2.0)
    q[:, :, 4:] *= 2.0 ** (-14 if source == torch.float16 else -20)
    lens = [150, 61]
    got = fp4.decode_attention(q, make_cache(kv, 160, device), 2, max_seqlen=150, causal=True,
                               seqlens=torch.tensor(lens, dtype=torch.int32, device=device))
    stored = oracle.rounded(wide(kv))
    assert (np.abs(stored[..., 1, :, :]) == 65536).any()
    want = oracle.attend(wide(q), stored, lens, True)
    for h in range(2):
        own = slice(4 * h, 4 * h + 4)
        tol = attend_tolerance(wide(q)[:, :, own], stored[:, :, :, h:h + 1], want[:, :, own], torch.float16)
        # (two sums of values that nearly cancel, in halves of fp16's smallest step too)
        assert (np.abs(wide(got)[:, :, own] - want[:, :, own]) <= tol + 2.0 ** -25).all()


def test_a_long_row_at_far_offsets(device):
    """A sequence whose rows lie beyond 4 GiB of the cache's start."""
    heads, d, n = 8, 128, 300
    capacity = (1 << 32) // fp4.row_bytes(heads, d) + 400
    cache = torch.empty((2, capacity, fp4.row_bytes(heads, d)), dtype=torch.uint8, device=device)
    kv = randn((1, n, 2, heads, d), 4, torch.bfloat16, device)
    start = capacity - n
    fp4.store_kv(cache[1:], kv, position_bias=start)
    assert same(fp4.load_kv(cache[1:], n, heads, d, torch.bfloat16, position_bias=start), oracle.rounded(wide(kv)))
    q = randn((1, 1, 32, d), 5, torch.bfloat16, device)
    got = fp4.decode_attention(q, cache[1:, start:], heads, max_seqlen=n, seqlen_bias=n)
    # the same rows through lengths that span the whole cache: zeros before them
    cache[1, :start] = 0
    long = fp4.decode_attention(q, cache[1:], heads, max_seqlen=capacity, seqlen_bias=capacity)
    stored = oracle.rounded(wide(kv))
    want = oracle.attend(wide(q), stored, [n])
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, torch.bfloat16)).all()
    # zero keys score 0 and hold zero values: they only add their count to the sum
    k = np.repeat(stored[0, :, 0].transpose(1, 0, 2), 4, axis=0)
    p = np.exp(np.einsum("hnd,hd->hn", k, wide(q)[0, 0]) * d ** -0.5)
    v = np.repeat(stored[0, :, 1].transpose(1, 0, 2), 4, axis=0)
    want = np.einsum("hn,hnd->hd", p, v) / (p.sum(-1) + start)[:, None]
    assert np.abs(wide(long)[0, 0] - want).max() <= 2.0 ** -8 * np.abs(want).max() + 2.0 ** -12 * np.abs(want).max()


# ---------------------------------------------------------------- products ---


def linear_tolerance(x, w, want, dtype):
    """Half a step of the type, and the fp32 sum's: k products, each within
    2^-24 of the sum of magnitudes."""
    return torch.finfo(dtype).eps / 2 * np.abs(want) + x.shape[-1] * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T) + 1e-30


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 32), (1, 16, 128), (2, 17, 96), (3, 250, 544), (16, 64, 2048), (17, 33, 160),
                                      (33, 50, 1056), (64, 128, 512), (65, 15, 64), (130, 129, 256), (300, 260, 320),
                                      # every kernel, tile and split: whole and ragged shares of the inner dimension
                                      (1, 41, 2080), (1, 33, 4128), (1, 30, 8224), (1, 18, 12288), (1, 17, 12320),
                                      (2, 19, 2048), (2, 35, 4064), (2, 21, 8192), (2, 18, 8224), (3, 18, 1056),
                                      (9, 40, 4128), (16, 33, 9216), (20, 8200, 96), (32, 8192, 1088), (17, 8193, 4160),
                                      (40, 8192, 160), (64, 8195, 1056), (50, 8192, 4128), (20, 100, 3200),
                                      (60, 70, 5152), (128, 200, 4096), (193, 140, 2080), (257, 300, 1056)])
def test_linear(device, dtype, rows, n, k):
    x = randn((rows, k), rows + n, dtype, device)
    w = fp4.quantize(randn((n, k), n + k, torch.float32, device, k ** -0.5))
    values = wide(fp4.dequantize(w, torch.float32))
    want = wide(x) @ values.T
    got = fp4.linear(x, w)
    assert (np.abs(wide(got) - want) <= linear_tolerance(wide(x), values, want, dtype)).all()
    assert torch.equal(got, fp4.linear(x, w))  # no order left to chance
    if rows > 1:  # a token's product does not depend on its neighbours
        skewed = torch.zeros((rows, k + 3), dtype=dtype, device=device)[:, 3:]
        skewed.copy_(x)
        assert torch.equal(fp4.linear(skewed, w), got)


# rows, n and k on either side of a prompt's tiles, of a step of 128 and of the
# splits; the largest tiles; inner dimensions below a step
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(65, 127, 128), (64 + 63, 129, 160), (128, 1, 224), (129, 257, 192), (320, 128, 1056),
                                      (321, 256, 416), (383, 257, 128), (330, 15, 2080), (70, 33, 96), (200, 40, 32),
                                      (4000, 4090, 160)])
def test_linear_of_a_prompt(device, dtype, rows, n, k):
    test_linear(device, dtype, rows, n, k)


@pytest.mark.parametrize("rows", [70, 400])
def test_a_prompt_with_a_far_power_in_the_last_step(device, rows):
    k, n = 416, 300
    x = randn((rows, k), 1, torch.float16, device)
    w = fp4.quantize(randn((n, k), 2, torch.float32, device))
    w.powers[7, 12], w.powers[299, 9], w.powers[260, 0] = 95, 100, 103
    values = wide(fp4.dequantize(w, torch.float32))
    want = wide(x) @ values.T
    assert (np.abs(wide(fp4.linear(x, w)) - want) <= linear_tolerance(wide(x), values, want, torch.float16)).all()
    w.powers[5, 12] = 255
    got = fp4.linear(x, w)
    assert torch.isnan(got[:, 5]).all() and torch.isfinite(got).sum() == rows * (n - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 40, 150])
def test_linear_with_far_powers_and_nan(device, dtype, rows):
    k, n = 384, 70
    x = randn((rows, k), 1, dtype, device)
    w = fp4.quantize(randn((n, k), 2, torch.float32, device))
    w.powers[3] = 90                # 2^-37, below what fp16 holds
    w.powers[5, 2] = 150            # 2^23, above it
    w.powers[6, :] = 0              # 2^-127
    w.powers[40, 7] = 255           # NaN
    values = wide(fp4.dequantize(w, torch.float32))
    got = wide(fp4.linear(x, w))
    assert np.isnan(got[:, 40]).all()
    keep = np.arange(n) != 40
    want = wide(x) @ values[keep].T
    with np.errstate(over="ignore"):
        want = torch.from_numpy(want).to(dtype).double().numpy() if dtype == torch.float16 else want
    tol = linear_tolerance(wide(x), values[keep], np.where(np.isfinite(want), want, 0), dtype)
    tol = tol + (2.0 ** -11 * np.abs(np.where(np.isfinite(want), want, 0)) + 2.0 ** -25 if dtype == torch.float16 else 0)
    big = ~np.isfinite(want)  # past fp16's range
    got = got[:, keep]
    assert np.array_equal(got[big], want[big]) and (np.abs(got[~big] - want[~big]) <= tol[~big]).all()


def test_linear_of_a_token_that_is_not_finite(device):
    x = randn((20, 64), 1, torch.float16, device)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    w = fp4.quantize(randn((40, 64), 2, torch.float32, device))
    got = fp4.linear(x, w)
    bad = ~torch.isfinite(got).all(-1)
    assert bad[3] and bad[4] and bad.sum() == 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 300), (2, 300), (3, 300), (20, 300), (40, 300), (100, 300), (400, 300), (4000, 4090)])
def test_an_infinite_activation_against_far_powers(device, dtype, rows, n):
    """Its product with a block that fp16 does not hold is an infinity, and no
    other block's zeros turn that, or an infinity beside them, into NaN."""
    k = 416
    x = randn((rows, k), 1, dtype, device)
    x[rows // 2, 70], x[rows - 1, 130] = float("inf"), -float("inf")
    w = fp4.quantize(randn((n, k), 2, torch.float32, device))
    w.codes.bitwise_or_(0x22)  # no element is zero
    w.powers[7, 2], w.powers[8, 4], w.powers[299, 2], w.powers[33, 12] = 95, 150, 100, 90
    values = wide(fp4.dequantize(w, torch.float32))
    finite = np.where(np.isfinite(wide(x)), wide(x), 0)
    want = finite @ values.T
    with np.errstate(invalid="ignore"):
        want += np.where(wide(x)[:, 70:71] == np.inf, np.inf * values[:, 70], 0)
        want += np.where(wide(x)[:, 130:131] == -np.inf, -np.inf * values[:, 130], 0)
    got, fine = wide(fp4.linear(x, w)), np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    fine &= np.abs(want) < 60000  # (within fp16, rounded)
    tol = linear_tolerance(finite, values, np.where(fine, want, 0), dtype)
    assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all()


@pytest.mark.parametrize("rows", [1, 3, 20, 50, 100, 200])
def test_linear_of_a_nan_with_a_small_payload(device, rows):
    """Its upper half alone would read as an infinity."""
    x = randn((rows, 64), 1, torch.float32, device)
    x.view(torch.int32)[rows - 1, 5] = 0x7F800001
    got = fp4.linear(x, fp4.quantize(randn((40, 64), 2, torch.float32, device)))
    assert torch.isnan(got[rows - 1]).all() and torch.isfinite(got[:rows - 1]).all()


# ----------------------------------------------------------- log-probabilities ---


def check_logprobs(logits, tokens, top):
    got = logprobs.token_logprobs(logits, tokens, top)
    x = wide(logits)
    vocab = x.shape[1]
    lp, entropy, ids, best = oracle.logprobs(x, tokens.cpu().numpy(), top)
    with np.errstate(all="ignore"):
        u = x - x.max(-1, keepdims=True)
        w = np.exp(u)
        mean = np.where(w > 0, np.where(w > 0, u, 0) ** 2 * w, 0).sum(-1) / w.sum(-1)  # E (x - m)^2
    mean = np.nan_to_num(mean)
    # sums: a lane's chain, then the lanes'; an exponential: its argument's rounding
    chain = (vocab / 256 + 32) * 2.0 ** -23

    def near(a, b, slack):
        a, fine = wide(a), np.isfinite(b)
        assert np.array_equal(a[~fine], b[~fine], equal_nan=True)
        assert (np.abs(a[fine] - b[fine]) <= (slack * np.ones_like(b))[fine] + 2.0 ** -22 * np.abs(b[fine])).all()

    slack = (chain + 2.0 ** -21) * (1 + mean)
    near(got.logprob, lp, slack)
    near(got.entropy, entropy, slack)
    if top:
        assert np.array_equal(got.top_ids.cpu().numpy(), ids)
        near(got.top_logprobs, best, slack[:, None])
    else:
        assert got.top_ids is None and got.top_logprobs is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (2, 64, 64), (5, 300, 5), (2, 8185, 20), (3, 8192, 3),
                                            (1, 32000, 5), (2, 50257, 64), (4, 16385, 0), (1100, 9001, 4)])
def test_logprobs(device, dtype, rows, vocab, top):
    logits = randn((rows, vocab), vocab, dtype, device, 3.0)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1)).to(device)
    check_logprobs(logits, tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1000, 20001])
def test_logprobs_of_rows_that_strain_it(device, dtype, vocab):
    rows = [torch.zeros(vocab), torch.arange(vocab) * (60000.0 / vocab), -torch.arange(vocab) * 0.01,
            torch.full((vocab,), -float("inf")), torch.zeros(vocab), torch.randn(vocab), torch.randn(vocab),
            torch.full((vocab,), torch.finfo(dtype).min), torch.randn(vocab), torch.full((vocab,), -0.0)]
    rows[4][:vocab - 1] = -float("inf")           # one token left
    rows[5][vocab // 2], rows[6][17] = float("nan"), float("inf")
    rows[8][: vocab - 3] = -float("inf")          # fewer than `top` left
    rows[9][1::2] = 0.0                           # -0 and 0 are equal
    logits = torch.stack(rows).to(dtype).to(device)
    tokens = torch.tensor([0, vocab - 1, -100, 3, vocab - 1, 5, 17, 2, 0, vocab]).to(device)
    check_logprobs(logits, tokens, 20)


# rows in one part and in several, on either side of the border between them, and
# of the most parts that each `top` allows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(2, 49137, 5), (2, 49152, 5), (3, 60001, 20), (1, 131100, 5), (2, 131072, 64),
                                            (2, 70000, 0), (1, 140000, 1), (40, 50001, 9), (1100, 49200, 2)])
def test_logprobs_of_long_vocabularies(device, dtype, rows, vocab, top):
    test_logprobs(device, dtype, rows, vocab, top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_of_long_rows_that_strain_it(device, dtype):
    test_logprobs_of_rows_that_strain_it(device, dtype, 60001)


def test_logprobs_of_strided_rows(device):
    base = randn((7, 12000), 3, torch.bfloat16, device)
    tokens = torch.tensor([5, 0, 7, 11, 2, 9, 4], device=device)
    for start, n in ((1, 9001), (3, 500), (0, 11999)):
        check_logprobs(base[:, start:start + n], tokens, 8)
    check_logprobs(base[2:3, 7:11007], tokens[:1], 64)
    stacked = logprobs.token_logprobs(base[:6].view(2, 3, 12000), tokens[:6].view(2, 3), 3)
    flat = logprobs.token_logprobs(base[:6], tokens[:6], 3)
    assert torch.equal(stacked.logprob.view(-1), flat.logprob) and stacked.top_ids.shape == (2, 3, 3)
    assert logprobs.token_logprobs(base[0, ::1]).entropy.shape == ()
    assert logprobs.token_logprobs(base[:0], tokens[:0], 3).top_ids.shape == (0, 3)


def narrow(rows, vocab, live, dtype, device, step=0.0):
    """Random logits with all but `live` neighbours ruled out (0: none, sorted);
    with ``step`` of few values, so that many are equal."""
    x = randn((rows, vocab), live, torch.float32, device, 3.0)
    if step:
        x = (x / step).round() * step
    if not live:
        return x.sort(-1).values.to(dtype)
    place = torch.arange(vocab, device=device)
    first = torch.arange(rows, device=device)[:, None] * (vocab - live) // max(1, rows - 1)
    return x.masked_fill((place < first) | (place >= first + live), -float("inf")).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,live,top,step", itertools.product((32000, 9001, 128000), (0, 257, 608, 3001), (20, 64), (0.0, 1.0, 20.0)))
def test_logprobs_of_narrow_masks(device, dtype, vocab, live, top, step):
    logits = narrow(3, vocab, live, dtype, device, step)
    if live == 608:
        logits[1, (vocab - live) // 2 + 100] = float("nan")
        logits[2, vocab - 300:] = float("nan")
    if not live:
        logits[2, 100:2100] = float("nan")  # more of them than can be ranked at once
    check_logprobs(logits, torch.tensor([5, vocab // 2, vocab - 1], device=device), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,live,step", [(1, 32000, 300, 0.0), (200, 32000, 600, 0.0), (1, 128000, 400, 0.0),
                                                  (1, 32000, 0, 0.0), (2, 32000, 400, 20.0)])
def test_narrow_masks_take_the_time_of_others(device, dtype, rows, vocab, live, step):
    """Within eight times the unmasked call's (it was 14 to 36 times where the
    largest was taken out ``top`` times over)."""
    def time(x):
        logprobs.token_logprobs(x, None, 20)
        rounds = []
        for _ in range(7):  # the least of them: what else the machine does is not timed
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(10):
                logprobs.token_logprobs(x, None, 20)
            end.record()
            end.synchronize()
            rounds.append(start.elapsed_time(end))
        return min(rounds)

    whole = randn((rows, vocab), 3, dtype, device, 3.0)
    assert time(narrow(rows, vocab, live, dtype, device, step)) <= 8 * time(whole)


def test_logprobs_of_a_padded_vocabulary(device):
    base = randn((2, 3, 9100), 3, torch.bfloat16, device)
    tokens = torch.tensor([[5, 0, 7], [11, 2, 9]], device=device)
    got = logprobs.token_logprobs(base[..., :9001], tokens, 4)
    want = logprobs.token_logprobs(base[..., :9001].contiguous(), tokens, 4)
    assert got.top_ids.shape == (2, 3, 4) and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------ streams and graphs ---


def test_a_step_on_another_stream_and_in_a_graph(device):
    """A decode step as it is used: product, append with attention, product,
    scores; eagerly, on a side stream, and replayed three times as a graph with
    eager work between the replays."""
    heads, hq, d, hidden, vocab = 2, 8, 64, 512, 9000
    wq = fp4.quantize(randn(((hq + 2 * heads) * d, hidden), 1, torch.bfloat16, device, hidden ** -0.5))
    wo = fp4.quantize(randn((vocab, hq * d), 2, torch.bfloat16, device, 0.1))
    kv = randn((3, 400, 2, heads, d), 3, torch.bfloat16, device)
    x = randn((3, 1, hidden), 4, torch.bfloat16, device)
    lens = torch.tensor([5, 399, 130], dtype=torch.int32, device=device)

    def step(cache):
        qkv = fp4.linear(x, wq)
        q, new = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:].contiguous()
        out = fp4.decode_attention(q, cache, heads, max_seqlen=400, seqlens=lens, kv_new=new)
        logits = fp4.linear(out.flatten(2), wo)
        return [out, logits, *logprobs.token_logprobs(logits, logits.argmax(-1), 5)]

    def fresh():
        return make_cache(kv, 400, device)

    cache = fresh()
    want = [t.clone() for t in step(cache)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))

    captured = fresh()
    first = captured.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        result = step(captured)
    for _ in range(3):
        captured.copy_(first)
        for t in result:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, result))
        assert torch.equal(captured, cache)
        step(fresh())  # eager work between


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_path_in_a_graph(device, dtype):
    """Chunks taken out and read in four bits (their keys split, so that both
    join), products with blocks fp16 does not hold and prompts, and rows of logits that are
    ranked, filled and counted: three replays, with the same calls made eagerly between them."""
    heads, hq, d, t, n = 1, 4, 128, 110, 2900
    kv = randn((1, n, 2, heads, d), 1, dtype, device)
    cache = make_cache(kv, n + 9, device)
    q = randn((1, t, hq, d), 2, dtype, device, 2.0)
    lens = torch.tensor([n - 3], dtype=torch.int32, device=device)
    w = fp4.quantize(randn((300, 4512), 3, dtype, device, 0.02))
    w.powers[7, 2], w.powers[290, 140] = 95, 150
    xs = [randn((rows, 4512), rows, dtype, device) for rows in (1, 9, 40, 200)]
    xs[1][3, 70] = float("inf")
    logits = torch.cat((narrow(2, 32000, 300, dtype, device), narrow(2, 32000, 0, dtype, device),
                        narrow(2, 32000, 9, dtype, device), torch.zeros((2, 32000), dtype=dtype, device=device)))

    def calls():
        return [fp4.decode_attention(q, cache, heads, max_seqlen=n, seqlens=lens, causal=True),
                fp4.decode_attention(q[:, :5], cache, heads, max_seqlen=n, seqlens=lens, causal=True),
                *(fp4.linear(x, w) for x in xs), *logprobs.token_logprobs(logits, None, 20)[1:],
                *logprobs.token_logprobs(logits[:, :9000], None, 20)[1:]]

    want = calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = calls()
    for _ in range(3):
        for r in result:
            r.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(torch.nan_to_num(a.double(), 7.5, 8.5, 9.5), torch.nan_to_num(b.double(), 7.5, 8.5, 9.5))
                   for a, b in zip(want, result))
        calls()  # eager work between


# --------------------------------------------------- refusals on the device ---


def test_calls_refuse_what_they_would_misread(device):
    x = randn((4, 64), 1, torch.float16, device)
    w = fp4.quantize(x)
    cache = fp4.kv_cache(2, 8, 2, 64, device)
    q = randn((2, 1, 4, 64), 1, torch.float16, device)
    empty = fp4.Fp4Tensor(w.codes[:, :0].contiguous(), w.powers[:, :0].contiguous())
    for call in (lambda: fp4.quantize(torch.zeros(128, device=device)[::2]),
                 lambda: fp4.linear(torch.zeros(128, device=device, dtype=torch.float16)[::2], w),
                 lambda: fp4.linear(x[:, :0], empty),
                 lambda: fp4.store_kv(cache, torch.zeros(2, 1, 2, 2, 64, device=device), None, 1 << 32),
                 lambda: fp4.load_kv(cache, (1 << 32) + 1, 2, 64, torch.float16),
                 lambda: fp4.load_kv(cache, 4, 2, 64, torch.float16,
                                     out=torch.empty(2, 1, 2, 2, 64, device=device, dtype=torch.float16).expand(2, 4, 2, 2, 64)),
                 lambda: fp4.decode_attention(q, cache, 2, max_seqlen=(1 << 32) + 4),
                 lambda: fp4.decode_attention(q, cache, 2, max_seqlen=4, seqlen_bias=1 << 32),
                 lambda: fp4.decode_attention(q, cache, 2, max_seqlen=4, partition=1 << 32)):
        with pytest.raises(ValueError):
            call()


def test_products_and_scores_of_nothing(device):
    w = fp4.quantize(randn((6, 64), 1, torch.float16, device))
    assert fp4.linear(torch.zeros(0, 64, device=device, dtype=torch.float16), w).shape == (0, 6)
    none = fp4.Fp4Tensor(w.codes[:0], w.powers[:0])
    assert fp4.linear(torch.zeros(3, 64, device=device, dtype=torch.float16), none).shape == (3, 0)
    got = logprobs.token_logprobs(torch.zeros(0, 9, device=device), torch.zeros(0, dtype=torch.int64, device=device), 2)
    assert got.logprob.shape == got.entropy.shape == (0,) and got.top_ids.shape == (0, 2)
    assert fp4.quantize(torch.zeros(3, 0, device=device)).codes.shape == (3, 0)


def test_calls_of_two_streams_side_by_side(device):
    """The same calls at once on two streams, their workspaces their own."""
    kv = randn((2, 1500, 2, 2, 64), 1, torch.bfloat16, device)
    cache = make_cache(kv, 1500, device)
    qs = [randn((2, 1, 8, 64), 5 + i, torch.bfloat16, device) for i in range(2)]
    xs = [randn((5, 512), 8 + i, torch.bfloat16, device) for i in range(2)]
    logits = [randn((2, 40000), 3 + i, torch.bfloat16, device) for i in range(2)]
    w = fp4.quantize(randn((512, 512), 2, torch.bfloat16, device))

    def calls(i):
        return [fp4.decode_attention(qs[i], cache, 2, max_seqlen=1500, seqlen_bias=1500), fp4.linear(xs[i], w),
                *logprobs.token_logprobs(logits[i], None, 7)[1:]]

    want = [calls(0), calls(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(calls(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
