"""Refusals and layouts of the 8-bit pool's and the paged attention's entry
points, without a GPU: every argument error comes back as a status before any
launch, empty calls are no-ops, and the Python and C++ front ends refuse tensors
of the wrong kind."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

import yllang_b200 as yl
from test_abi import _c_layout
from yllang_b200 import _abi


@pytest.mark.parametrize("struct,cls", [("yl_quant_pool", _abi.QuantPool), ("yl_quant_store_args", _abi.QuantStoreArgs),
                                        ("yl_quant_load_args", _abi.QuantLoadArgs),
                                        ("yl_paged_attention_args", _abi.PagedAttentionArgs)])
def test_struct_layout_matches_header(tmp_path, struct, cls):
    names = [f for f, _ in cls._fields_]
    c = _c_layout(tmp_path, struct, names)
    assert c["size"] == ctypes.sizeof(cls)
    for f in names:
        assert c[f] == getattr(cls, f).offset, f


def _set(a, kw):
    for k, v in kw.items():
        if k.startswith("pool_"):
            setattr(a.pool, k[5:], v)
        else:
            setattr(a, k, v)
    return a


def _pool(a):
    return _set(a, dict(pool_k_codes=0x10000, pool_v_codes=0x20000, pool_k_scale=0x3000, pool_v_scale=0x4000,
                        pool_page_stride=8192, pool_slot_stride=128, pool_head_stride=2048, pool_scale_page_stride=4,
                        pool_scale_head_stride=1, pool_num_pages=10, pool_page_size=16, pool_num_heads=4,
                        pool_head_dim=128, pool_num_layers=1))


def _store(**kw):
    base = dict(k=0x50000, v=0x60000, kv_indptr=0x7000, kv_indices=0x8000, kv_last_page_len=0x9000, qo_indptr=0xA000,
                kv_indices_capacity=10, num_tokens=4, k_row_stride=1024, v_row_stride=1024, batch_size=2, dtype=0)
    return _set(_pool(_abi.QuantStoreArgs()), {**base, **kw})


POOL_ERRORS = [
    (dict(pool_num_layers=0), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_page_size=0), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_num_heads=0), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_num_pages=0), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_head_dim=96), _abi.YL_ERR_UNSUPPORTED),
    (dict(pool_num_pages=1 << 27), _abi.YL_ERR_UNSUPPORTED),  # 2^31 slots
    (dict(pool_num_pages=1 << 31), _abi.YL_ERR_UNSUPPORTED),
    (dict(pool_num_layers=1 << 30), _abi.YL_ERR_UNSUPPORTED),
    (dict(pool_num_heads=2 ** 31 - 1), _abi.YL_ERR_UNSUPPORTED),
    (dict(pool_k_codes=0), _abi.YL_ERR_NULL_ARG),
    (dict(pool_v_scale=0), _abi.YL_ERR_NULL_ARG),
    (dict(pool_slot_stride=64), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_scale_head_stride=0), _abi.YL_ERR_BAD_SIZE),
    (dict(pool_v_codes=0x20004), _abi.YL_ERR_ALIGNMENT),
    (dict(pool_page_stride=8196), _abi.YL_ERR_ALIGNMENT),
    (dict(pool_k_scale=0x3002), _abi.YL_ERR_ALIGNMENT),
]


@pytest.mark.parametrize("kw,status", POOL_ERRORS + [
    (dict(batch_size=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(num_tokens=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(kv_indices_capacity=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(dtype=2), _abi.YL_ERR_BAD_SIZE),
    (dict(v=0), _abi.YL_ERR_NULL_ARG),
    (dict(qo_indptr=0), _abi.YL_ERR_NULL_ARG),
    (dict(k_row_stride=512), _abi.YL_ERR_BAD_SIZE),
    (dict(v_row_stride=1032), _abi.YL_ERR_ALIGNMENT),
    (dict(k=0x50008), _abi.YL_ERR_ALIGNMENT),
    (dict(pool_num_layers=2, k_layer_stride=-16), _abi.YL_ERR_BAD_SIZE),
    (dict(num_tokens=1 << 31), _abi.YL_ERR_UNSUPPORTED),
])
def test_quant_store_rejects_bad_arguments_on_host(kw, status):
    assert _abi.kv_quant_store_raw(_store(**kw), None) == status
    assert _abi.last_error().startswith("yl_kv_quant_store")


def _load(**kw):
    base = dict(k_out=0x50000, v_out=0x60000, slots=0x7000, num_tokens=4, k_row_stride=1024, v_row_stride=1024,
                slot_is_int64=1, dtype=1)
    return _set(_pool(_abi.QuantLoadArgs()), {**base, **kw})


@pytest.mark.parametrize("kw,status", POOL_ERRORS + [
    (dict(num_tokens=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(slot_is_int64=2), _abi.YL_ERR_BAD_SIZE),
    (dict(dtype=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(k_out=0), _abi.YL_ERR_NULL_ARG),
    (dict(slots=0), _abi.YL_ERR_NULL_ARG),
    (dict(slots=0x7004), _abi.YL_ERR_ALIGNMENT),
    (dict(pool_slot_stride=136), _abi.YL_ERR_ALIGNMENT),  # 16 bytes here, 8 for the store
    (dict(v_row_stride=1000), _abi.YL_ERR_BAD_SIZE),
    (dict(num_tokens=1 << 28), _abi.YL_ERR_UNSUPPORTED),
])
def test_quant_load_rejects_bad_arguments_on_host(kw, status):
    assert _abi.kv_quant_load_raw(_load(**kw), None) == status
    assert _abi.last_error().startswith("yl_kv_quant_load")


def _attend(**kw):
    base = dict(q=0x10000, o=0x20000, k_cache=0x30000, v_cache=0x40000, k_scale=0x5000, v_scale=0x6000,
                kv_indptr=0x7000, kv_indices=0x8000, kv_last_page_len=0x9000, qo_indptr=0xA000, workspace=0xB0000,
                workspace_bytes=1 << 40, q_row_stride=8192, q_head_stride=256, o_row_stride=8192, o_head_stride=256,
                page_stride=16384, slot_stride=128, head_stride=2048, scale_page_stride=8, scale_head_stride=1,
                kv_indices_capacity=10, num_pages=10, num_tokens=4, batch_size=2, num_q_heads=32, num_kv_heads=8,
                head_dim=128, page_size=16, dtype=0, kv_dtype=1, sm_scale=0.1)
    return _set(_abi.PagedAttentionArgs(), {**base, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(batch_size=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(num_tokens=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(num_tokens=1 << 31), _abi.YL_ERR_UNSUPPORTED),
    (dict(num_tokens=1 << 30), _abi.YL_ERR_UNSUPPORTED),  # times the group
    (dict(dtype=2), _abi.YL_ERR_BAD_SIZE),
    (dict(kv_dtype=2), _abi.YL_ERR_BAD_SIZE),
    (dict(head_dim=80), _abi.YL_ERR_UNSUPPORTED),
    (dict(num_kv_heads=0), _abi.YL_ERR_BAD_SIZE),
    (dict(num_q_heads=30), _abi.YL_ERR_BAD_SIZE),
    (dict(num_q_heads=32768, num_kv_heads=32768), _abi.YL_ERR_UNSUPPORTED),
    (dict(page_size=0), _abi.YL_ERR_BAD_SIZE),
    (dict(window=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(sinks=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(max_new_len=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(sm_scale=0.0), _abi.YL_ERR_BAD_SIZE),
    (dict(sm_scale=float("nan")), _abi.YL_ERR_BAD_SIZE),
    (dict(sm_scale=float("inf")), _abi.YL_ERR_BAD_SIZE),
    (dict(kv_indices_capacity=-1), _abi.YL_ERR_BAD_SIZE),
    (dict(num_pages=0), _abi.YL_ERR_BAD_SIZE),
    (dict(q=0), _abi.YL_ERR_NULL_ARG),
    (dict(kv_indices=0), _abi.YL_ERR_NULL_ARG),
    (dict(v_scale=0), _abi.YL_ERR_NULL_ARG),
    (dict(workspace=0), _abi.YL_ERR_NULL_ARG),
    (dict(workspace_bytes=100), _abi.YL_ERR_BAD_SIZE),
    (dict(workspace=0xB0008), _abi.YL_ERR_ALIGNMENT),
    (dict(q_head_stride=128), _abi.YL_ERR_BAD_SIZE),
    (dict(head_stride=64), _abi.YL_ERR_BAD_SIZE),
    (dict(kv_dtype=0, slot_stride=128), _abi.YL_ERR_BAD_SIZE),
    (dict(scale_page_stride=0), _abi.YL_ERR_BAD_SIZE),
    (dict(o=0x20008), _abi.YL_ERR_ALIGNMENT),
    (dict(page_stride=16392), _abi.YL_ERR_ALIGNMENT),
])
def test_paged_attention_rejects_bad_arguments_on_host(kw, status):
    assert _abi.paged_attention_raw(_attend(**kw), None) == status
    assert _abi.last_error().startswith("yl_paged_attention")


@pytest.mark.parametrize("call,make,names", [
    (_abi.kv_quant_store_raw, _store, ["kv_indptr", "kv_indices", "kv_last_page_len", "qo_indptr", "error_word"]),
    (_abi.kv_quant_load_raw, _load, ["error_word"]),
    (_abi.paged_attention_raw, _attend, ["kv_indptr", "kv_indices", "kv_last_page_len", "qo_indptr", "k_scale", "v_scale",
                                         "error_word"]),
], ids=["store", "load", "attention"])
def test_words_off_their_alignment_are_refused(call, make, names):
    """A kernel would fault on them."""
    for name in names:
        assert call(make(**{name: 0x9002}), None) == _abi.YL_ERR_ALIGNMENT, name
        assert "4-byte aligned" in _abi.last_error()


@pytest.mark.parametrize("kw", [dict(pool_layer_stride=0), dict(pool_scale_layer_stride=0)])
def test_layers_that_a_store_writes_lie_apart(kw):
    """An expanded pool would be written by all layers at once; broadcast rows are read."""
    apart = dict(pool_num_layers=2, pool_layer_stride=1 << 20, pool_scale_layer_stride=64)
    assert _abi.kv_quant_store_raw(_store(**{**apart, **kw}), None) == _abi.YL_ERR_BAD_SIZE
    assert "apart" in _abi.last_error()


@pytest.mark.parametrize("kw", [dict(k_layer_stride=0), dict(v_layer_stride=0)])
def test_layers_that_a_load_writes_lie_apart(kw):
    apart = dict(pool_num_layers=2, k_layer_stride=1 << 20, v_layer_stride=1 << 20)
    assert _abi.kv_quant_load_raw(_load(**{**apart, **kw}), None) == _abi.YL_ERR_BAD_SIZE
    assert "apart" in _abi.last_error()


def test_empty_calls_are_noops_without_device():
    L = yl.lib()
    assert _abi.kv_quant_store_raw(_store(num_tokens=0, k=0), None) == _abi.YL_OK
    assert _abi.kv_quant_store_raw(_store(batch_size=0, k=0), None) == _abi.YL_OK
    assert _abi.kv_quant_load_raw(_load(num_tokens=0, slots=0), None) == _abi.YL_OK
    assert _abi.paged_attention_raw(_attend(num_tokens=0, q=0), None) == _abi.YL_OK
    assert _abi.paged_attention_raw(_attend(batch_size=0, q=0), None) == _abi.YL_OK
    for f in (L.yl_kv_quant_store, L.yl_kv_quant_load, L.yl_paged_attention):
        assert f(None, None) == _abi.YL_ERR_NULL_ARG
    assert L.yl_paged_attention_workspace(None) == _abi.YL_ERR_NULL_ARG


def test_workspace_bytes():
    """No pointers needed; enough for both halves of every CTA's unfinished results."""
    one = _abi.paged_attention_workspace_raw(_attend(q=0, workspace=0, max_new_len=1, num_q_heads=8))
    many = _abi.paged_attention_workspace_raw(_attend(q=0, workspace=0))
    assert 0 < one < many < 1 << 27
    assert _abi.paged_attention_workspace_raw(_attend(head_dim=5)) == _abi.YL_ERR_UNSUPPORTED


def test_launch_without_device_reports_cuda_error():
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    assert _abi.kv_quant_store_raw(_store(), None) == _abi.YL_ERR_CUDA
    assert _abi.kv_quant_load_raw(_load(), None) == _abi.YL_ERR_CUDA
    assert _abi.paged_attention_raw(_attend(), None) == _abi.YL_ERR_CUDA


def _index(B=2):
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    return yl.BatchIndex(i(B + 1), i(4), i(B), i(B + 1), None)


def test_front_ends_refuse_host_tensors_and_wrong_kinds():
    pool = yl.quant_kv_pool(4, 16, 2, 64, device="cpu")
    rows = torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(yl.PanicError, match="CUDA"):
        yl.store_kv_cache_quant(rows, rows, pool, _index())
    with pytest.raises(yl.PanicError, match="CUDA"):
        yl.load_kv_cache_quant(pool, torch.zeros(3, dtype=torch.int64))
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(yl.PanicError, match="CUDA"):
        yl.paged_attention(q, q, q, _index())
    with pytest.raises(yl.PanicError, match="Hq"):
        yl.paged_attention(q[0], q, q, _index())
    with pytest.raises(yl.PanicError, match="CUDA"):
        yl.paged_attention_workspace(q, q, q, _index())


def test_front_ends_refuse_a_stream_of_another_device():
    """Such a call would otherwise run on the current stream of the tensors' device."""
    stream = SimpleNamespace(device=torch.device("cuda", 1))
    pool = yl.quant_kv_pool(4, 16, 2, 64, device="cpu")
    rows = torch.zeros(3, 128, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: yl.store_kv_cache_quant(rows, rows, pool, _index(), stream=stream),
                 lambda: yl.load_kv_cache_quant(pool, torch.zeros(3, dtype=torch.int64), stream=stream),
                 lambda: yl.paged_attention(q, q, q, _index(), stream=stream)):
        with pytest.raises(yl.PanicError, match="stream is on cuda:1"):
            call()


def test_quant_pool_layout():
    """Views of head-major pages: the tokens that share a scale are contiguous."""
    pool = yl.quant_kv_pool(5, 16, 3, 64, num_layers=2, device="cpu")
    assert pool.k.shape == (2, 5, 16, 3, 64) and pool.k.stride() == (5 * 3 * 16 * 64, 3 * 16 * 64, 64, 16 * 64, 1)
    assert pool.k.dtype == torch.float8_e4m3fn and pool.k_scale.shape == (2, 5, 3)
    one = pool.layer(1)
    assert one.k.shape == (5, 16, 3, 64) and one.k.data_ptr() == pool.k[1].data_ptr() and one.v_scale.shape == (5, 3)
    C = yl.load_extension()
    assert {"StoreKVCacheQuant", "LoadKVCacheQuant", "PagedAttention", "PagedAttentionWorkspace"} <= set(dir(C))
    assert C.DeviceErrorNames(0x28000) == _abi.deverr_names(0x28000) == "NONFINITE|SCALE"
    made = C.MakeQuantKVPool(5, 16, 3, 64, num_layers=2, device=torch.device("cpu"))
    for a, b in zip(made, pool):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
        assert torch.equal(a.float(), b.float())
    assert C.MakeQuantKVPool(5, 16, 3, 64, device=torch.device("cpu"))[2].shape == (5, 3)
    with pytest.raises(RuntimeError, match="positive"):
        C.MakeQuantKVPool(5, 0, 3, 64, device=torch.device("cpu"))
