"""The four-bit and scoring calls without a GPU: the oracle pinned by values
written out by hand, the ABI's structure, and every refusal before a launch."""
import ctypes
import subprocess

import numpy as np
import pytest
import torch

from hexgen2_amd import _lib, fp4, logprobs, mha
from hexgen2_amd.engine import Engine
from hexgen2_amd.generation import InferenceParams
from hexgen2_amd.llama import LlamaHost, LlamaShape, read_config
from hexgen2_amd.run import parse_args
from oracle import mx_oracle as oracle
from tests.test_abi import ROOT

GOLDEN = ROOT / "tests" / "golden"


def test_oracle_rounds_to_the_nearest_even_code():
    x = np.zeros(32)
    x[:15] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.2500001, 0.2499, 0.76, -1.24, 2.51, 3.49, -5.01]
    codes, powers = oracle.quantize(x)
    assert powers.tolist() == [127]
    want = [6, 0, 1, 1, 2, 2, 4, 4, -0.5, 0, 1, -1, 3, 3, -6]
    assert oracle.values(codes, powers)[:15].tolist() == want


@pytest.mark.parametrize("most,power", [(6.0, 0), (6.0001, 1), (3.0, -1), (3.01, 0), (12.0, 1), (1.5 * 2.0 ** -30, -32),
                                        (1e-40, -125), (3e38, 126), (0.0, 0)])
def test_oracle_power_is_the_smallest_that_holds_the_block(most, power):
    x = np.full(32, most / 7)
    x[11] = -most
    assert (oracle.quantize(x)[1] - 127).tolist() == [power]


def test_oracle_marks_blocks_that_are_not_finite():
    x = np.ones((3, 32))
    x[0, 3], x[1, 31] = np.inf, np.nan
    codes, powers = oracle.quantize(x)
    assert powers[:, 0].tolist() == [255, 255, 125]  # 1 = 4 * 2^-2
    assert np.isnan(oracle.values(codes, powers)[:2]).all() and (oracle.values(codes, powers)[2] == 1).all()


def test_oracle_rows_round_trip():
    rng = np.random.default_rng(0)
    kv = rng.standard_normal((3, 2, 2, 64))
    rows = oracle.rows(kv)
    assert rows.shape[-1] == fp4.row_bytes(2, 64) == 144
    assert np.array_equal(oracle.row_values(rows, 2, 64), oracle.rounded(kv))


def test_oracle_logprobs_by_hand():
    lp, entropy, ids, best = oracle.logprobs([[0.0, 0.0, -np.inf, 0.0], [-np.inf] * 4, [1.0, np.nan, 2.0, 0.0]],
                                             [2, 1, -1], 2)
    assert lp[0] == -np.inf and lp[1] == -np.inf and lp[2] == 0
    assert entropy[:2] == pytest.approx([np.log(3), 0]) and np.isnan(entropy[2])
    assert ids.tolist() == [[0, 1], [0, 1], [1, 2]]
    assert best[0] == pytest.approx([-np.log(3)] * 2)


def test_params_layout_matches_c(tmp_path):
    fields = [f[0] for f in _lib.MxAttendParams._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hexkv.h"\nint main(void){\n'
                   'printf("%zu\\n", sizeof(hexkv_mx_attend_params));\n'
                   + "".join(f'printf("%zu\\n", offsetof(hexkv_mx_attend_params, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.MxAttendParams)] + [getattr(_lib.MxAttendParams, f).offset for f in fields]


E, R, U, W = _lib.HEXKV_EINVAL, _lib.HEXKV_ERANGE, _lib.HEXKV_EUNSUPPORTED, _lib.HEXKV_EWORKSPACE
ADDRESS = 1 << 12  # never dereferenced: every call below is refused


def rows_call(**change):
    a = dict(kv=ADDRESS, kv_bs=512, kv_ps=256, kv_hs=128, cache=ADDRESS, c_bs=144 * 8, c_ps=144, capacity=8, batch=2,
             seqlen=3, heads=2, d=64, dtype=1, positions=None, bias=0)
    a.update(change)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), E), (dict(batch=-1), E), (dict(seqlen=-1), E), (dict(heads=0), E), (dict(d=48), U), (dict(d=0), U),
    (dict(d=2048), U), (dict(kv=None), E), (dict(cache=None), E), (dict(capacity=0), E), (dict(c_ps=128), E),
    (dict(c_ps=152, c_bs=152 * 8), E), (dict(cache=ADDRESS + 8), E), (dict(c_bs=144 * 7), E), (dict(kv=ADDRESS + 1), E),
    (dict(bias=6), R), (dict(bias=-1), R), (dict(batch=1, seqlen=9), R),
    (dict(batch=1 << 20, seqlen=1 << 11, capacity=1 << 11, c_bs=144 << 11), R),
])
@pytest.mark.parametrize("name", ["hexkv_mx_store", "hexkv_mx_load"])
def test_row_calls_refuse(name, change, code):
    a = rows_call(**change)
    rows, cache = [a["kv"], a["kv_bs"], a["kv_ps"], a["kv_hs"]], [a["cache"], a["c_bs"], a["c_ps"], a["capacity"]]
    lead = rows + cache if name == "hexkv_mx_store" else cache + rows
    rc = getattr(_lib.load(), name)(*lead, a["batch"], a["seqlen"], a["heads"], a["d"], a["dtype"], a["positions"],
                                    a["bias"], None)
    assert rc == code and _lib.load().hexkv_last_error()


@pytest.mark.parametrize("args,code", [
    ((ADDRESS, 64, ADDRESS, ADDRESS, 4, 48, 1), E), ((ADDRESS, 64, ADDRESS, ADDRESS, -1, 64, 1), E),
    ((ADDRESS, 64, ADDRESS, ADDRESS, 4, 64, 7), E), ((None, 64, ADDRESS, ADDRESS, 4, 64, 1), E),
    ((ADDRESS, 64, ADDRESS + 2, ADDRESS, 4, 64, 1), E), ((ADDRESS, 64, ADDRESS, ADDRESS, 1 << 31, 64, 1), R),
    ((ADDRESS, 64, ADDRESS, ADDRESS, 0, 64, 1), 0), ((None, 0, None, None, 5, 0, 1), 0)])
def test_matrix_calls_refuse(args, code):
    x, stride, codes, powers, rows, width, dtype = args
    lib = _lib.load()
    assert lib.hexkv_mx_quantize(x, stride, codes, powers, rows, width, dtype, None) == code
    assert lib.hexkv_mx_dequantize(codes, powers, x, stride, rows, width, dtype, None) == code


def attend_params(**change):
    p = _lib.MxAttendParams(dtype=1, batch=2, q_len=1, q_heads=4, kv_heads=2, head_dim=64, softmax_scale=0.125, q=ADDRESS,
                            q_batch_stride=256, q_row_stride=256, cache=ADDRESS, cache_batch_bytes=144 * 300,
                            cache_row_bytes=144, capacity=300, out=ADDRESS, out_batch_stride=256, out_row_stride=256,
                            seqlen_bias=9, max_seqlen=300)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(dtype=5), E), (dict(q_len=0), E), (dict(kv_heads=3), E), (dict(head_dim=16), U), (dict(head_dim=96), U),
    (dict(max_seqlen=301), R), (dict(max_seqlen=-1), R), (dict(partition=48), E), (dict(partition=-32), E),
    (dict(partition=1 << 17), E), (dict(softmax_scale=0.0), E), (dict(softmax_scale=float("inf")), E),
    (dict(softmax_scale=float("nan")), E), (dict(q_len=2, kv_new=ADDRESS), E), (dict(cache_row_bytes=128), E),
    (dict(cache_row_bytes=152), E), (dict(cache_batch_bytes=144 * 299), E), (dict(cache_row_bytes=1 << 25, batch=1), E),
    (dict(q=None), E), (dict(cache=None), E), (dict(out=None), E), (dict(cache=ADDRESS + 8), E), (dict(out=ADDRESS + 1), E),
    (dict(kv_new=ADDRESS + 8), E), (dict(partition=32), W), (dict(batch=1 << 20, q_len=1 << 10), R)])
def test_attention_refuses(change, code):
    p = attend_params(**change)
    assert _lib.load().hexkv_mx_attend(ctypes.byref(p), None, 0, None) == code
    assert _lib.load().hexkv_last_error()


@pytest.mark.parametrize("change", [
    # nine pairs take the places of sixteen: 9/16 of 2^24 workgroups and a few more
    dict(batch=9, q_len=(1 << 24) + 16, q_heads=1, kv_heads=1, head_dim=32, max_seqlen=32),
    # a workgroup per row in the join of 17 partitions, eight rows a workgroup in that of two
    dict(batch=1, q_len=1 << 23, q_heads=1, kv_heads=1, head_dim=32, max_seqlen=17 * 32, partition=32),
    dict(batch=1, q_len=1 << 26, q_heads=1, kv_heads=1, head_dim=32, max_seqlen=64, partition=32)])
def test_attention_refuses_launches_of_too_many_lanes(change):
    """(With room enough said to be at an address that is never read: the refusal comes first.)"""
    p = attend_params(dtype=0, capacity=1 << 10, cache_row_bytes=48, cache_batch_bytes=48 << 10, **change)
    assert _lib.load().hexkv_mx_attend(ctypes.byref(p), ADDRESS, 1 << 62, None) == R
    assert b"2^32 lanes" in _lib.load().hexkv_last_error()


def test_attention_refuses_a_small_workspace_and_null_params():
    lib, p = _lib.load(), attend_params(partition=32)
    need = lib.hexkv_mx_attend_workspace_bytes(ctypes.byref(p))
    assert need >= 2 * 4 * 10 * 66 * 4  # a partial output, maximum and sum per row and partition
    assert lib.hexkv_mx_attend(ctypes.byref(p), ADDRESS, need - 1, None) == W
    assert lib.hexkv_mx_attend(ctypes.byref(p), ADDRESS + 4, need, None) == E
    assert lib.hexkv_mx_attend(None, None, 0, None) == E
    p.batch = 0
    assert lib.hexkv_mx_attend(ctypes.byref(p), None, 0, None) == 0


@pytest.mark.parametrize("args,code", [
    ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, 4, 8, 64, 9), E), ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, 4, 8, 48, 1), E),
    ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, 4, 8, 0, 1), E), ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, -4, 8, 64, 1), E),
    ((None, 64, ADDRESS, ADDRESS, ADDRESS, 4, 8, 64, 1), E), ((ADDRESS, 64, ADDRESS + 4, ADDRESS, ADDRESS, 4, 8, 64, 1), E),
    ((ADDRESS + 1, 64, ADDRESS, ADDRESS, ADDRESS, 4, 8, 64, 1), E), ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, 1 << 21, 8, 64, 1), R),
    ((ADDRESS, 64, ADDRESS, ADDRESS, ADDRESS, 0, 8, 64, 1), 0)])
def test_linear_refuses(args, code):
    assert _lib.load().hexkv_mx_linear(*args, None, 0, None) == code


def logprob_call(**change):
    a = dict(logits=ADDRESS, stride=1000, rows=3, vocab=1000, dtype=1, tokens=ADDRESS, top=4, lp=ADDRESS, entropy=ADDRESS,
             values=ADDRESS, ids=ADDRESS, ws=None, size=0)
    a.update(change)
    return _lib.load().hexkv_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=4), E), (dict(rows=-1), E), (dict(vocab=0), E), (dict(vocab=(1 << 30) + 1), E), (dict(top=-1), E),
    (dict(top=65), E), (dict(top=9, vocab=8), E), (dict(rows=1 << 19), R), (dict(logits=None), E), (dict(lp=None), E),
    (dict(ids=None), E), (dict(values=None), E), (dict(logits=ADDRESS + 1), E), (dict(tokens=ADDRESS + 4), E),
    (dict(vocab=64000), W), (dict(vocab=64000, ws=ADDRESS, size=8), W), (dict(rows=0), 0)])
def test_logprobs_refuse(change, code):
    assert logprob_call(**change) == code


def test_python_refuses_what_is_not_on_the_gpu():
    x = torch.zeros(4, 64)
    w = fp4.Fp4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8))
    cache = torch.zeros(1, 8, 144, dtype=torch.uint8)
    for call in (lambda: fp4.quantize(x), lambda: fp4.dequantize(w, torch.float16), lambda: fp4.linear(x, w),
                 lambda: fp4.store_kv(cache, torch.zeros(1, 1, 2, 2, 64)),
                 lambda: fp4.load_kv(cache, 1, 2, 64, torch.float16),
                 lambda: fp4.decode_attention(torch.zeros(1, 1, 4, 64), cache, 2, max_seqlen=4),
                 lambda: logprobs.token_logprobs(torch.zeros(2, 8))):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_row_bytes():
    assert [fp4.row_bytes(*g) for g in ((8, 128), (1, 128), (4, 64), (32, 128), (1, 32))] == [1088, 144, 272, 4352, 48]
    for bad in ((0, 64), (2, 48), (2, 0)):
        with pytest.raises(ValueError):
            fp4.row_bytes(*bad)


def test_four_bit_caches_through_the_module_calls():
    assert mha.inference_cache(2, 9, 2, 64, torch.float16, "cpu", kv_bits=4).shape == (2, 9, 144)
    assert mha.inference_cache(2, 9, 2, 64, torch.float16, "cpu").shape == (2, 9, 2, 2, 64)
    for bits, ft, d in ((8, False, 64), (4, True, 64), (4, False, 48)):
        with pytest.raises(ValueError):
            mha.inference_cache(2, 9, 2, d, torch.float16, "cpu", ft, bits)
    params = InferenceParams(9, kv_bits=4)
    with pytest.raises(ValueError, match="HIP device"):
        mha._update_kv_cache(torch.zeros(1, 2, 2, 2, 64), params, 0)
    assert InferenceParams(9).kv_bits == 16


@pytest.mark.parametrize("bits", [{"kv_bits": 8}, {"weight_bits": 2}, {"kv_bits": 0}])
def test_engine_refuses_other_widths(bits):
    with pytest.raises(ValueError, match="16 bits"):
        Engine(GOLDEN / "fixture_seed17", "native", "cpu", "float16", **bits)


def test_host_refuses_other_widths():
    shape = LlamaShape.from_config(read_config(GOLDEN / "fixture_seed17"))
    with pytest.raises(ValueError, match="16 bits"):
        LlamaHost(shape, {}, "cpu", torch.float16, weight_bits=8)


def test_pilot_arguments(capsys):
    base = ["--model-dir", "m", "--trace", "t", "--output", "o"]
    args = parse_args(base)
    assert (args.kv_bits, args.weight_bits, args.logprobs) == (16, 16, False)
    args = parse_args(base + ["--kv-bits", "4", "--weight-bits", "4", "--logprobs"])
    assert (args.kv_bits, args.weight_bits, args.logprobs) == (4, 4, True)
    with pytest.raises(SystemExit):
        parse_args(base + ["--kv-bits", "8"])


def test_a_row_of_strided_elements_is_refused():
    assert fp4._matrix_rows(torch.zeros(64), "x") == 64
    assert fp4._matrix_rows(torch.zeros(3, 128)[:, :64], "x") == 128
    for t in (torch.zeros(128)[::2], torch.zeros(64, 3).t(), torch.zeros(2, 3, 128)[..., :64]):
        with pytest.raises(ValueError, match="contiguous"):
            fp4._matrix_rows(t, "x")


def test_sizes_past_32_bits_are_refused():
    assert [fp4._int32(v, "x") for v in (-(1 << 31), (1 << 31) - 1)] == [-(1 << 31), (1 << 31) - 1]
    for value in (1 << 31, 1 << 32, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="32 bits"):
            fp4._int32(value, "x")
    p = attend_params(max_seqlen=(1 << 31) - 1, capacity=1 << 31, batch=1)
    assert _lib.load().hexkv_mx_attend(ctypes.byref(p), None, 0, None) == R


def test_shapes_past_32_bits_are_refused():
    """Sizes that ctypes would wrap to a smaller call (views of one element: nothing is allocated)."""
    long, bits = (1 << 32) + 64, torch.float16
    one = torch.zeros(1, dtype=bits)
    with pytest.raises(ValueError, match="32 bits"):
        logprobs._form(torch.Size((1, long)), (long, 1), bits, 2)
    with pytest.raises(ValueError, match="32 bits"):
        fp4._linear_form(torch.Size((1, long)), (long, 1), bits, torch.Size((4, long // 2)), torch.Size((4, long // 32)))
    with pytest.raises(ValueError, match="32 bits"):
        fp4._rows_form(one.expand(1, long, 2, 1, 32).shape, (0, 0, 0, 32, 1), bits)
    with pytest.raises(ValueError, match="32 bits"):
        fp4._attend_form(one.expand(1, long, 1, 32), torch.zeros(1, 4, 48, dtype=torch.uint8), 1, None, None, False, None, 0)
    with pytest.raises(ValueError, match="32 bits"):
        fp4._matrix_size((1, long))
    assert logprobs._form(torch.Size((2, 9)), (16, 1), bits, 2)[:3] == (2, 9, 16)


def test_logits_of_any_dims_whose_rows_lie_at_one_stride():
    x = torch.zeros(4, 3, 5, 20)
    for t, want in ((x, (60, 20, 20)), (x[..., :17], (60, 17, 20)), (x[1, 2, 3], (1, 20, 20)), (x[:, :, 2:3, :9], (12, 9, 100)),
                    (x[:, 1, 2, :1], (4, 1, 300)), (x[:0, ..., :9], (0, 9, 9)), (x[:1, :1, :, 3:], (5, 17, 20)),
                    (x[0, 0, 0].expand(6, 20), (6, 20, 0)), (torch.zeros(20, 7).t()[:, :1], (7, 1, 1))):
        assert logprobs._form(t.shape, t.stride(), t.dtype, 0)[:3] == want
    for t in (x[:, :2], x[..., ::2], x.transpose(0, 1), x[:, :, :2, :9], x[:, :1].expand(4, 3, 5, 20)):
        with pytest.raises(ValueError, match="logits rows"):
            logprobs._form(t.shape, t.stride(), t.dtype, 0)


def test_parameters_without_the_field_keep_16_bits():
    class Plain:  # the reference's own fields
        max_sequence_len, max_batch_size, sequence_len_offset, batch_size_offset = 9, 1, 0, 0
        fused_ft_kernel, lengths_per_sample, key_value_memory_dict = False, None, {}
    assert mha._kv_bits(Plain()) == 16 and mha._kv_bits(InferenceParams(9, kv_bits=4)) == 4
    with pytest.raises(ValueError, match="HIP device"):
        mha._update_kv_cache(torch.zeros(1, 2, 2, 2, 64), Plain(), 0)
    assert Plain.key_value_memory_dict[0].shape == (1, 9, 2, 2, 64)
