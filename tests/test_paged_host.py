"""Paged caches without a GPU: the oracle and the rotary frequencies pinned by
values written out by hand, the ABI's structures, and every refusal before a launch."""
import ctypes
import math
import subprocess

import numpy as np
import pytest
import torch

from hexgen2_amd import _lib, mha, paged, rotary
from hexgen2_amd.engine import Engine
from hexgen2_amd.generation import InferenceParams
from hexgen2_amd.llama import LlamaShape, read_config
from hexgen2_amd.run import parse_args
from oracle import kv_oracle, paged_oracle as oracle
from tests.test_abi import ROOT

GOLDEN = ROOT / "tests" / "golden"


# ---------------------------------------------------------------- oracle ---


def test_oracle_rotation_by_hand():
    x = np.array([[1.0, 2.0, 3.0, 4.0, 5.0]])
    f = [math.pi / 2, math.pi]  # a quarter and a half turn a position
    assert np.allclose(oracle.rotate(x, 1, f), [[-3, -2, 1, -4, 5]])
    assert np.allclose(oracle.rotate(x, 1, f, interleaved=True), [[-2, 1, -3, -4, 5]])
    assert np.allclose(oracle.rotate(x, 2, f, scale=0.5), [[-0.5, 1, -1.5, 2, 5]])


def test_oracle_append_places_rows():
    pages = np.zeros((3, 2, 2, 1, 2))
    qkv = np.arange(12.0).reshape(2, 6)  # q, k, v of one head of two
    q, got = oracle.append(qkv, pages, [[2, 1], [0, -1]], [3, -1], [0, 1, 2], 1, [])
    assert np.array_equal(q[0], [[0, 1]]) and np.isnan(q[1]).all()
    assert np.array_equal(got[1, 1], [[[2, 3]], [[4, 5]]]) and np.count_nonzero(got) == 4


def test_oracle_attention_matches_the_plain_caches():
    rng = np.random.default_rng(0)
    lens, size = [5, 9], 4
    tables = [[3, 1, -1], [0, 4, 2]]
    pages, q = rng.standard_normal((5, size, 2, 2, 8)), rng.standard_normal((4, 4, 8))
    starts = [3, 7]
    out, weight, reach = oracle.attend(q, pages, tables, starts, [0, 2, 4])
    cache = np.stack([np.stack([pages[t[p // size], p % size] if p < n else np.zeros((2, 2, 8)) for p in range(9)])
                      for t, n in zip(tables, lens)])
    for t in range(2):  # token t of both sequences, over starts + t + 1 keys
        want = kv_oracle.attend(q[[t, 2 + t]][:, None], cache, [4 + t, 8 + t])
        assert np.allclose(out[[t, 2 + t]], want[:, 0])
    assert (np.abs(out) <= weight + 1e-12).all() and (reach > 0).all()


def test_oracle_pack_round_trip():
    rng = np.random.default_rng(1)
    pages = rng.standard_normal((4, 2, 2, 1, 3))
    packed = oracle.pack(pages, [[2, 0], [3, -1]], [3, 1])
    assert np.array_equal(packed, np.stack([pages[2, 0], pages[2, 1], pages[0, 0], pages[3, 0]]))
    back = oracle.unpack(packed, np.zeros_like(pages), [[2, 0], [3, -1]], [3, 1])
    assert np.array_equal(back[2], pages[2]) and not back[1].any() and not back[0, 1].any() and not back[3, 1].any()


# ------------------------------------------------------------- frequencies ---


def test_plain_and_linear_frequencies():
    f, scale = rotary.frequencies(8, 10000.0)
    assert scale == 1 and f.dtype == torch.float32 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    f, scale = rotary.frequencies(8, 10000.0, {"type": "linear", "factor": 4})
    assert scale == 1 and torch.allclose(f, torch.tensor([0.25, 0.025, 0.0025, 0.00025]))
    assert rotary.frequencies(0)[0].shape == (0,)


def test_llama3_frequencies():
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 200}
    f, scale = rotary.frequencies(8, 10000.0, s)
    # turns over 200 positions: 31.8, 3.18, 0.318, 0.0318
    kept = (20 / (2 * math.pi) - 1) / 3
    assert scale == 1 and torch.allclose(f, torch.tensor([1.0, 0.1 * (kept + (1 - kept) / 8), 0.01 / 8, 0.001 / 8]))


def test_yarn_frequencies():
    s = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 200, "beta_fast": 20, "beta_slow": 2}
    f, scale = rotary.frequencies(8, 10000.0, s)
    # the pairs that make 20 and 2 turns lie at 0.20 and 1.20, so at 0 and 2
    assert scale == pytest.approx(0.1 * math.log(4) + 1)
    assert torch.allclose(f, torch.tensor([1.0, 0.1 * (0.5 + 0.5 / 4), 0.01 / 4, 0.001 / 4]))
    assert rotary.frequencies(8, 10000.0, dict(s, attention_factor=1.5))[1] == 1.5
    assert rotary.frequencies(8, 10000.0, dict(s, attention_factor=None, mscale=None))[1] == scale
    for more in (dict(mscale=0.7), dict(mscale_all_dim=1.0), dict(truncate=False), dict(attention_factor=-1.0)):
        with pytest.raises(ValueError, match="yarn"):
            rotary.frequencies(8, 10000.0, dict(s, **more))


@pytest.mark.parametrize("scaling,match", [({"rope_type": "dynamic", "factor": 2.0}, "dynamic"), ({"rope_type": "linear"}, "factor"),
                                           ({"rope_type": "llama3", "factor": 2.0}, "original_max_position"),
                                           ({"rope_type": "linear", "factor": 0}, "factor"),
                                           ({"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4, "high_freq_factor": 4,
                                             "original_max_position_embeddings": 10}, "above")])
def test_scalings_that_are_refused(scaling, match):
    with pytest.raises(ValueError, match=match):
        rotary.frequencies(64, 10000.0, scaling)


def test_model_settings_name_their_scaling():
    config = read_config(GOLDEN / "tiny_llama")
    assert LlamaShape.from_config(config).rope_scaling is None
    scaling = {"rope_type": "linear", "factor": 2.0}
    assert LlamaShape.from_config(dict(config, rope_scaling=scaling)).rope_scaling == scaling
    with pytest.raises(ValueError, match="longrope"):
        LlamaShape.from_config(dict(config, rope_scaling={"type": "longrope"}))


# ------------------------------------------------------------------- ABI ---


@pytest.mark.parametrize("c_name,mirror", [("hexkv_pool", _lib.Pool), ("hexkv_paged_batch", _lib.PagedBatch),
                                            ("hexkv_paged_append_params", _lib.PagedAppendParams),
                                            ("hexkv_paged_attend_params", _lib.PagedAttendParams)])
def test_struct_layouts_match_c(tmp_path, c_name, mirror):
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hexkv.h"\nint main(void){\n'
                   f'printf("%zu\\n", sizeof({c_name}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({c_name}, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    values = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert values == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


# Addresses that no call below gets as far as using.
QKV, Q, PAGES, TABLE = 1 << 20, 2 << 20, 1 << 30, 4 << 20


def pool(**changes):
    p = _lib.Pool(dtype=_lib.HEXKV_F16, kv_heads=2, head_dim=64, n_pages=8, page_size=16, page_stride=2 * 2 * 16 * 64,
                  pos_stride=64, kv_stride=16 * 64, head_stride=2 * 16 * 64)
    for k, v in changes.items():
        setattr(p, k, v)
    return p


def seqs(**changes):
    s = _lib.PagedBatch(tables=TABLE, table_stride=4, table_width=4, batch=2, starts=TABLE, cu_tokens=TABLE, tokens=6)
    for k, v in changes.items():
        setattr(s, k, v)
    return s


def append_params(**changes):
    p = _lib.PagedAppendParams(pool=pool(), seqs=seqs(), q_heads=4, qkv=QKV, qkv_stride=8 * 64, q=Q, q_stride=4 * 64,
                               pages=PAGES, inv_freq=TABLE, rotary_dim=64, interleaved=0, rotary_scale=1.0)
    for k, v in changes.items():
        setattr(p, k, v)
    return p


def attend_params(**changes):
    p = _lib.PagedAttendParams(pool=pool(), seqs=seqs(), q_heads=4, causal=1, softmax_scale=0.125, max_tokens=6, max_seqlen=60,
                               q=Q, q_stride=4 * 64, out=QKV, out_stride=4 * 64, pages=PAGES, partition=0)
    for k, v in changes.items():
        setattr(p, k, v)
    return p


COMMON = [
    (dict(pool=pool(dtype=7)), _lib.HEXKV_EINVAL, "dtype"),
    (dict(pool=pool(head_dim=48)), _lib.HEXKV_EUNSUPPORTED, "head_dim"),
    (dict(pool=pool(kv_heads=0)), _lib.HEXKV_EINVAL, "KV heads"),
    (dict(pool=pool(n_pages=0)), _lib.HEXKV_EINVAL, "page"),
    (dict(pool=pool(page_size=8)), _lib.HEXKV_EINVAL, "page_size"),
    (dict(pool=pool(page_size=48)), _lib.HEXKV_EINVAL, "page_size"),
    (dict(pool=pool(page_stride=1 << 30)), _lib.HEXKV_ERANGE, "2\\^30"),
    (dict(pool=pool(pos_stride=32)), _lib.HEXKV_EINVAL, "apart"),
    (dict(pool=pool(pos_stride=(1 << 26) + 8)), _lib.HEXKV_EINVAL, "apart"),
    (dict(pool=pool(kv_stride=1025)), _lib.HEXKV_EINVAL, "16 bytes"),
    (dict(pool=pool(head_stride=-64)), _lib.HEXKV_EINVAL, "16 bytes"),
    (dict(seqs=seqs(batch=-1)), _lib.HEXKV_EINVAL, "negative"),
    (dict(seqs=seqs(table_stride=3)), _lib.HEXKV_EINVAL, "overlap"),
    (dict(seqs=seqs(tables=None)), _lib.HEXKV_EINVAL, "tables"),
    (dict(seqs=seqs(starts=None)), _lib.HEXKV_EINVAL, "starts"),
    (dict(seqs=seqs(tokens=-1)), _lib.HEXKV_EINVAL, "negative"),
    (dict(seqs=seqs(tokens=5, cu_tokens=None)), _lib.HEXKV_EINVAL, "equal shares"),
    (dict(seqs=seqs(batch=0, tokens=5, cu_tokens=None)), _lib.HEXKV_EINVAL, "equal shares"),
    (dict(seqs=seqs(table_width=1 << 27, table_stride=1 << 27)), _lib.HEXKV_ERANGE, "2\\^30"),
    (dict(pages=PAGES + 8), _lib.HEXKV_EINVAL, "aligned"),
    (dict(pages=None), _lib.HEXKV_EINVAL, "null"),
]


def refused(call, code, match):
    import re
    lib = _lib.load()
    assert call(lib) == code, lib.hexkv_last_error()
    assert re.search(match, lib.hexkv_last_error().decode()), lib.hexkv_last_error()


@pytest.mark.parametrize("changes,code,match", COMMON + [
    (dict(q_heads=-1), _lib.HEXKV_EINVAL, "query heads"),
    (dict(rotary_dim=3), _lib.HEXKV_EINVAL, "rotary_dim"),
    (dict(rotary_dim=66), _lib.HEXKV_EINVAL, "rotary_dim"),
    (dict(qkv_stride=8 * 64 - 1), _lib.HEXKV_EINVAL, "overlap"),
    (dict(q_stride=4 * 64 - 1), _lib.HEXKV_EINVAL, "overlap"),
    (dict(inv_freq=None), _lib.HEXKV_EINVAL, "null"),
    (dict(q=QKV + 128), _lib.HEXKV_EINVAL, "q overlaps"),
    (dict(q=QKV, q_stride=4 * 64), _lib.HEXKV_EINVAL, "q overlaps"),
    (dict(qkv=PAGES + 4096), _lib.HEXKV_EINVAL, "pages overlap"),
    (dict(q=PAGES), _lib.HEXKV_EINVAL, "pages overlap"),
    (dict(seqs=seqs(tokens=1 << 24)), _lib.HEXKV_ERANGE, "2\\^24 tokens"),
])
def test_append_refuses(changes, code, match):
    refused(lambda lib: lib.hexkv_paged_append(ctypes.byref(append_params(**changes)), None), code, match)


@pytest.mark.parametrize("changes,code,match", COMMON + [
    (dict(q_heads=3), _lib.HEXKV_EINVAL, "query heads"),
    (dict(q_heads=0), _lib.HEXKV_EINVAL, "query heads"),
    (dict(softmax_scale=0.0), _lib.HEXKV_EINVAL, "softmax_scale"),
    (dict(softmax_scale=float("nan")), _lib.HEXKV_EINVAL, "softmax_scale"),
    (dict(softmax_scale=float("inf")), _lib.HEXKV_EINVAL, "softmax_scale"),
    (dict(max_seqlen=65), _lib.HEXKV_ERANGE, "max_seqlen"),
    (dict(max_seqlen=-1), _lib.HEXKV_ERANGE, "max_seqlen"),
    (dict(max_tokens=-1), _lib.HEXKV_EINVAL, "max_tokens"),
    (dict(q_stride=4 * 64 + 4), _lib.HEXKV_EINVAL, "aligned"),
    (dict(q=Q + 2), _lib.HEXKV_EINVAL, "aligned"),
    (dict(out_stride=100), _lib.HEXKV_EINVAL, "overlap"),
    (dict(partition=32), _lib.HEXKV_EINVAL, "multiple of 64"),
    (dict(partition=-64), _lib.HEXKV_EINVAL, "multiple of 64"),
    (dict(out=None), _lib.HEXKV_EINVAL, "null"),
    (dict(out=Q + 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q + 2 * 4 * 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q - 2 * 4 * 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q, out_stride=8 * 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q + 2 * 4 * 64 - 2, q_stride=8 * 64, out_stride=8 * 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q + 2 * 4 * 64 + 2, q_stride=8 * 64, out_stride=8 * 64), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=Q + 64, seqs=seqs(tokens=1, batch=1)), _lib.HEXKV_EINVAL, "rows of q"),
    (dict(out=PAGES), _lib.HEXKV_EINVAL, "overlaps the pages"),
    (dict(out=PAGES + 2 * 8 * 2 * 2 * 16 * 64 - 2), _lib.HEXKV_EINVAL, "overlaps the pages"),
    # sizes past the launch's: 2^31 rows, 2^24 workgroups
    (dict(pool=pool(kv_heads=1), q_heads=1 << 16, q_stride=64 << 16, out_stride=64 << 16, seqs=seqs(tokens=1 << 16), max_tokens=1 << 16),
     _lib.HEXKV_ERANGE, "rows"),
    (dict(pool=pool(kv_heads=1, dtype=_lib.HEXKV_F32), q_heads=1 << 10, q_stride=64 << 10, out_stride=64 << 10,
          seqs=seqs(tokens=1 << 19), max_tokens=1 << 19), _lib.HEXKV_ERANGE, "workgroups"),
])
def test_attention_refuses(changes, code, match):
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(attend_params(**changes)), None, 0, None), code, match)


def test_attention_refuses_a_missing_workspace():
    wide = dict(seqs=seqs(table_width=1024, table_stride=1024), max_seqlen=16384)
    lib = _lib.load()
    p = attend_params(**wide)
    need = lib.hexkv_paged_attend_workspace_bytes(ctypes.byref(p))
    assert need > 0
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), None, 0, None), _lib.HEXKV_EWORKSPACE, "workspace")
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), QKV, need - 1, None), _lib.HEXKV_EWORKSPACE, "workspace")
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), QKV + 4, need, None), _lib.HEXKV_EWORKSPACE, "workspace")
    for at in (Q, QKV, PAGES + 4096, Q - need + 16):
        refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), at, need, None), _lib.HEXKV_EINVAL, "workspace overlaps")
    assert lib.hexkv_paged_attend_workspace_bytes(ctypes.byref(attend_params())) == 0  # short rows are not split
    assert lib.hexkv_paged_attend_workspace_bytes(ctypes.byref(attend_params(max_seqlen=65))) == 0


def test_calls_without_work_do_nothing():
    lib = _lib.load()
    for changes in (dict(seqs=seqs(tokens=0)), dict(seqs=seqs(batch=0)), dict(seqs=seqs(batch=0, tokens=0, cu_tokens=None))):
        assert lib.hexkv_paged_append(ctypes.byref(append_params(**changes)), None) == 0
        assert lib.hexkv_paged_attend(ctypes.byref(attend_params(**changes)), None, 0, None) == 0
    assert lib.hexkv_paged_attend(ctypes.byref(attend_params(max_tokens=0)), None, 0, None) == 0


@pytest.mark.parametrize("name", ["hexkv_paged_pack", "hexkv_paged_unpack"])
@pytest.mark.parametrize("changes,code,match", [
    (dict(pool=pool(page_size=24)), _lib.HEXKV_EINVAL, "page_size"),
    (dict(layers=-1), _lib.HEXKV_EINVAL, "layer count"),
    (dict(lens=(65, 0)), _lib.HEXKV_ERANGE, "length 65"),
    (dict(lens=(-1, 0)), _lib.HEXKV_ERANGE, "length -1"),
    (dict(src=QKV + 4), _lib.HEXKV_EINVAL, "aligned"),
    (dict(dst=0), _lib.HEXKV_EINVAL, "null"),
    (dict(tables=None), _lib.HEXKV_EINVAL, "tables"),
    (dict(stride=2), _lib.HEXKV_EINVAL, "overlap"),
])
def test_handoff_refuses(name, changes, code, match):
    a = dict(pool=pool(), src=QKV, dst=PAGES, layers=1, tables=TABLE, stride=4, lens=(10, 3))
    a.update(changes)
    ptr = lambda x: (ctypes.c_void_p * 1)(x)  # noqa: E731
    refused(lambda lib: getattr(lib, name)(ctypes.byref(a["pool"]), ptr(a["src"]), ptr(a["dst"]), a["layers"], a["tables"],
                                           a["stride"], 4, 2, (ctypes.c_int64 * 2)(*a["lens"]), None), code, match)


@pytest.mark.parametrize("name", ["hexkv_paged_pack", "hexkv_paged_unpack"])
def test_handoff_refuses_more_workgroups_than_a_launch_has(name):
    ptr = lambda x: (ctypes.c_void_p * 1)(x)  # noqa: E731
    p = pool(kv_heads=1, head_dim=16, pos_stride=16, kv_stride=16 * 16, head_stride=0, page_stride=2 * 16 * 16)
    refused(lambda lib: getattr(lib, name)(ctypes.byref(p), ptr(QKV), ptr(PAGES), 1, TABLE, 1 << 23, 1 << 23, 1,
                                           (ctypes.c_int64 * 1)(1 << 26), None), _lib.HEXKV_ERANGE, "2\\^22 workgroups")


# -------------------------------------------------------- Python's checks ---


def tensors(dtype=torch.float16):
    pages = torch.zeros((4, 2, 2, 16, 64), dtype=dtype).transpose(1, 3)
    return dict(pages=pages, tables=torch.zeros((2, 3), dtype=torch.int32), starts=torch.zeros(2, dtype=torch.int32),
                cu=torch.tensor([0, 1, 5], dtype=torch.int32))


def test_cpu_tensors_are_refused():
    t = tensors()
    with pytest.raises(ValueError, match="HIP device"):
        paged.append(torch.zeros(5, 8 * 64, dtype=torch.float16), t["pages"], t["tables"], t["starts"], q_heads=4)
    with pytest.raises(ValueError, match="HIP device"):
        paged.attention(torch.zeros(5, 4, 64, dtype=torch.float16), t["pages"], t["tables"], t["starts"], max_seqlen=8)
    with pytest.raises(ValueError, match="HIP device"):
        paged.pack_live([t["pages"]], t["tables"], [1, 2])


def test_pool_layout():
    pool = paged.kv_pages(3, 16, 2, 64, torch.float16, "cpu")
    assert pool.shape == (3, 16, 2, 2, 64) and pool.stride() == (4096, 64, 1024, 2048, 1)
    assert paged.kv_pages(3, 16, 2, 64, torch.float16, "cpu", layers=5).shape == (5, 3, 16, 2, 2, 64)
    assert [paged.pages_for(n, 16) for n in (0, 1, 16, 17)] == [0, 1, 1, 2]
    p = paged._check_pages(pool, True)
    assert (p.n_pages, p.page_size, p.kv_heads, p.head_dim, p.pos_stride) == (3, 16, 2, 64, 64)
    one = paged._check_pages(torch.zeros((1, 16, 2, 1, 64)), True)
    assert (one.page_stride, one.head_stride) == (0, 0)


@pytest.mark.parametrize("make,match", [
    (lambda t: t["pages"][..., :32, :].unsqueeze(0), "pages must be"),
    (lambda t: t["pages"].int(), "float16"),
    (lambda t: t["pages"].transpose(3, 4), "contiguous"),
    (lambda t: t["pages"][:, :1].expand(4, 16, 2, 2, 64), "share elements"),
    (lambda t: t["pages"][:0], "pages must be"),
])
def test_pools_that_are_refused(make, match):
    with pytest.raises(ValueError, match=match):
        paged._check_pages(make(tensors()), True)


def append_form(t, qkv=None, q_heads=4, inv_freq=None, out=None, **changes):
    t = dict(t, **changes)
    qkv = torch.zeros(5, 8 * 64, dtype=torch.float16) if qkv is None else qkv
    return paged._append_form(qkv, t["pages"], t["tables"], t["starts"], t["cu"], q_heads, inv_freq, False, 1.0, out)


def test_append_form_and_its_refusals():
    t = tensors()
    p, shape = append_form(t, inv_freq=torch.ones(16))
    assert shape == (5, 4, 64) and (p.rotary_dim, p.seqs.tokens, p.seqs.batch, p.seqs.table_width) == (32, 5, 2, 3)
    assert append_form(t, torch.zeros(1, 5, 512, dtype=torch.float16))[1] == (1, 5, 4, 64)
    assert append_form(t, torch.zeros(5, 256, dtype=torch.float16), q_heads=0)[1] == (5, 0, 64)
    for changes, match in ((dict(qkv=torch.zeros(5, 500, dtype=torch.float16)), "qkv must be"), (dict(qkv=torch.zeros(5, 512)), "qkv must be"),
                           (dict(q_heads=-1), "qkv must be"), (dict(inv_freq=torch.ones(33)), "inv_freq"),
                           (dict(inv_freq=torch.ones(16).double()), "inv_freq"), (dict(tables=t["tables"].long()), "tables must be"),
                           (dict(tables=t["tables"].t()), "tables must be"), (dict(starts=t["starts"][:1]), "starts must be"),
                           (dict(starts=t["starts"].long()), "starts must be"), (dict(cu=t["cu"][:2]), "cu_tokens must be"),
                           (dict(out=torch.zeros(5, 4, 32, dtype=torch.float16)), "out must be"),
                           (dict(qkv=torch.zeros(10, 512, dtype=torch.float16)[::2].view(5, 512).expand(5, 512).t().contiguous().t()), "contiguous")):
        with pytest.raises(ValueError, match=match):
            append_form(t, **changes)


def test_attention_form_and_its_refusals():
    t = tensors()
    q = torch.zeros(5, 4, 64, dtype=torch.float16)

    def form(q=q, out=None, max_tokens=4, partition=0, **changes):
        u = dict(t, **changes)
        return paged._attend_form(q, u["pages"], u["tables"], u["starts"], u["cu"], max_tokens, True, None, out, partition)[0]

    p = form()
    assert (p.seqs.tokens, p.q_heads, p.q_stride, p.max_tokens) == (5, 4, 256, 4) and p.softmax_scale == 0.125
    assert form(q=torch.zeros(10, 6, 64, dtype=torch.float16)[::2, :4]).q_stride == 768
    for changes, match in ((dict(q=q.float()), "q must be"), (dict(q=q[:, :3]), "q must be"), (dict(q=q[..., :32]), "q must be"),
                           (dict(q=q[:, :0]), "q must be"), (dict(out=q[:4]), "out must"), (dict(max_tokens=1 << 31), "32 bits"),
                           (dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous")):
        with pytest.raises(ValueError, match=match):
            form(**changes)


def test_engine_and_pilot_options():
    for options, match in ((dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"),
                           (dict(page_size=16, kv_bits=4), "data type"), (dict(prefill_chunk=4), "page_size"),
                           (dict(page_size=16, prefill_chunk=-1), "chunks")):
        with pytest.raises(ValueError, match=match):
            Engine(GOLDEN / "tiny_llama", "native", "cuda", "float16", **options)
    args = parse_args(["--model-dir", "m", "--trace", "t", "--output", "o", "--page-size", "32", "--prefill-chunk", "64"])
    assert (args.page_size, args.prefill_chunk) == (32, 64)
    args = parse_args(["--model-dir", "m", "--trace", "t", "--output", "o"])
    assert (args.page_size, args.prefill_chunk) == (0, 0)


def test_steps_of_paged_caches():
    params = InferenceParams(max_sequence_len=40, max_batch_size=3, batch_size_offset=1, page_size=16)
    tables, starts, bound = mha.paged_sequences(params, 2, 5, torch.device("cpu"))
    assert tables.tolist() == [[3, 4, 5], [6, 7, 8]] and starts.tolist() == [0, 0] and bound == 5
    params.sequence_len_offset, params.lengths_per_sample = 7, torch.tensor([1, 2, 3], dtype=torch.int32)
    _, starts, bound = mha.paged_sequences(params, 2, 1, torch.device("cpu"))
    assert starts.tolist() == [2, 3] and bound == 8
    params.sequence_len_offset = 40
    with pytest.raises(AssertionError):
        mha.paged_sequences(params, 2, 1, torch.device("cpu"))
    for changes in (dict(kv_bits=4), dict(fused_ft_kernel=True)):
        with pytest.raises(ValueError, match="paged caches"):
            mha.paged_sequences(InferenceParams(max_sequence_len=40, page_size=16, **changes), 1, 1, torch.device("cpu"))
