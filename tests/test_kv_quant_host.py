"""Host side of the 8-bit cache and the rotary forms: configuration, frequency tables, pool shapes, and the refusals of
the C entry points and of the tensor wrappers (none needs a GPU: every check fails before any launch)."""

import ctypes
import math

import pytest
import torch

from forgeserve_b200 import ModelConfig, PagedKVPool
from forgeserve_b200 import _lib as L
from forgeserve_b200 import ops
from forgeserve_b200.engine import check_kv_dtype
from forgeserve_b200.model import RopeTables, precompute_rope, rope_frequencies, rope_tables

F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from forgeserve_b200 import build
        build.build()
    return L.load()


def test_config_rotary_fields():
    assert "rope_layout" not in ModelConfig().to_dict() and ModelConfig().rotary_width == 16
    cfg = ModelConfig(rope_layout="interleaved", rotary_dim=8, rope_scaling={"kind": "linear", "factor": 2.0})
    assert ModelConfig(**cfg.to_dict()) == cfg and cfg.rotary_width == 8
    for bad in (dict(rope_layout="both"), dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=18),
                dict(rope_scaling={"kind": "other", "factor": 2}), dict(rope_scaling="linear"), dict(rope_scaling={"kind": "linear"}),
                dict(rope_scaling={"kind": "linear", "factor": 0.5}),
                dict(rope_scaling={"kind": "linear", "factor": 2, "beta_fast": 1}),
                dict(rope_scaling={"kind": "by_parts", "factor": 2}),
                dict(rope_scaling={"kind": "by_parts", "factor": 2, "original_max_len": 64, "beta_slow": 40}),
                dict(rope_scaling={"kind": "by_parts", "factor": 2, "original_max_len": 64, "attn_factor": 0})):
        with pytest.raises(ValueError):
            ModelConfig(**bad)


def test_rope_tables():
    """The plain form keeps the reference's tables; each scaling against its definition, pair by pair."""
    cfg = ModelConfig()
    t = RopeTables(cfg)
    c, s = precompute_rope(cfg.head_dim, cfg.max_seq_len, cfg.rope_theta)
    assert torch.equal(t.cos, c) and torch.equal(t.sin, s)
    rd, theta, f, n = 64, 10000.0, 8.0, 2048
    base = [theta ** (-2 * i / rd) for i in range(rd // 2)]
    lin, a = rope_frequencies(rd, theta, {"kind": "linear", "factor": f})
    assert a == 1.0 and lin.tolist() == pytest.approx([b / f for b in base], rel=1e-12)
    ntk, _ = rope_frequencies(rd, theta, {"kind": "ntk", "factor": f})
    assert ntk[0] == 1.0 and float(ntk[-1]) == pytest.approx(base[-1] / f, rel=1e-12)
    parts, a = rope_frequencies(rd, theta, {"kind": "by_parts", "factor": f, "original_max_len": n, "attn_factor": 1.5})
    assert a == 1.5
    for b, got in zip(base, parts.tolist()):
        turns = n * b / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 31))
        assert got == pytest.approx(b * (keep + (1 - keep) / f), rel=1e-12)
        assert b / f * 0.999 <= got <= b * 1.001
    assert float(rope_frequencies(2, theta, {"kind": "ntk", "factor": f})[0]) == 1 / f
    cos, sin = rope_tables(rd, 100001, theta, {"kind": "by_parts", "factor": f, "original_max_len": n, "attn_factor": 1.5})
    assert cos.shape == (100001, 32) and cos.dtype == torch.float32
    for i in (0, 5, 31):
        assert float(cos[100000, i]) == pytest.approx(1.5 * math.cos(100000 * float(parts[i])), abs=2e-7)
        assert float(sin[100000, i]) == pytest.approx(1.5 * math.sin(100000 * float(parts[i])), abs=2e-7)


def test_quantised_pool_shapes():
    cfg = ModelConfig()
    pool = PagedKVPool(cfg, 6, 4, dtype=F8)
    assert pool.quantized and pool.k[0].dtype == F8 and pool.k[0].shape == (6, 4, 4, 16)
    assert pool.k_scale[3].shape == pool.v_scale[0].shape == (6, 4, 4) and pool.k_scale[0].dtype == torch.float32
    d = pool.views(torch.tensor([[1, 2]]), torch.tensor([[0]]))[2].descriptor()
    assert isinstance(d, L.KVQuantDesc) and d.k_scale == pool.k_scale[2].data_ptr()
    assert (d.cache.block_stride, d.cache.head_stride, d.scale_block_stride, d.scale_head_stride) == (256, 64, 16, 4)
    plain = PagedKVPool(cfg, 6, 4)
    assert not plain.quantized and not hasattr(plain, "k_scale")
    check_kv_dtype(None, torch.bfloat16)
    check_kv_dtype(F8, torch.bfloat16)
    with pytest.raises(ValueError):
        check_kv_dtype(torch.float16, torch.bfloat16)


def test_descriptor_refusals():
    k = torch.zeros(4, 2, 8, 16).to(F8)
    s, t = torch.zeros(4, 2, 8), torch.zeros(1, 2, dtype=torch.int64)
    ops.quant_paged_desc(k, k, s, s, t)
    ops.quant_paged_desc(k[:, :1], k[:, :1], s[:, :1], s[:, :1], t)
    for args in ((k.float(), k, s, s, t), (k, k, s.half(), s, t), (k, k[:3], s, s, t), (k, k, s[:, :1], s, t),
                 (k, k, s, s, t[0]), (k[..., :8], k[..., :8], s, s, t), (k[:, :, ::2], k[:, :, ::2], s[:, :, ::2], s[:, :, ::2], t)):
        with pytest.raises((TypeError, ValueError)):
            ops.quant_paged_desc(*args)


def test_wrappers_refuse_cpu_tensors():
    k = torch.zeros(4, 2, 8, 16).to(F8)
    s, t = torch.zeros(4, 2, 8), torch.zeros(1, 2, dtype=torch.int64)
    d = ops.quant_paged_desc(k, k, s, s, t)
    with pytest.raises(RuntimeError, match="CUDA kernels only"):
        ops.rotary_kv_write(torch.zeros(1, 8 * 16), None, None, torch.zeros(1, dtype=torch.int64), d, 1, 1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA kernels only"):
        ops.kv_dequant(d, 1, 8, 2, 16, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA kernels only"):
        ops.attention_decode_quant(torch.zeros(1, 64), d, 8, torch.zeros(1, dtype=torch.int64), torch.zeros(1, 64), 1, 4,
                                   2, 16)


def quant_desc(p=4096, **kw):
    base = dict(k=p, v=p, table=p, table_stride=8, table_cols=8, block_size=16, block_stride=2 * 16 * 128,
                head_stride=16 * 128, num_blocks=4)
    base.update(kw)
    return L.KVQuantDesc(L.KVCacheDesc(**base), p, p, 32, 16)


P = ctypes.c_void_p(4096)          # never dereferenced: the checks fail before any launch


def rotary_args(**kw):
    a = dict(qkv=P, ld=1024, q_out=P, ldq=1024, cos=P, sin=P, rows=64, rd=128, inter=0, pos=P, kv=None, B=1, T=1, nh=4,
             nkv=2, hd=128, base=0, from_pos=1, dtype=L.FS_BF16, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("quant", [False, True])
def test_rotary_write_refusals(lib, quant):
    fn = lib.fs_rotary_kv_write_quant if quant else lib.fs_rotary_kv_write
    desc = quant_desc() if quant else quant_desc().cache
    ref = ctypes.byref(desc)
    for kw, word in ((dict(qkv=None), b"NULL"), (dict(pos=None), b"NULL"), (dict(q_out=None), b"NULL"),
                     (dict(cos=None), b"tables"), (dict(rows=0), b"tables"), (dict(rd=3), b"rotary_dim"),
                     (dict(rd=130), b"rotary_dim"), (dict(rd=-2), b"rotary_dim"), (dict(hd=0), b"head_dim"),
                     (dict(hd=127), b"head_dim"), (dict(hd=514), b"head_dim"), (dict(nkv=0), b"head counts"),
                     (dict(nh=-1), b"head counts"), (dict(ld=1000), b"qkv row stride"), (dict(ldq=500), b"q_out row"),
                     (dict(dtype=7), b"dtype"), (dict(from_pos=0, base=-1), b"slot_base"),
                     (dict(T=1 << 40), b"too many"), (dict(B=1 << 20, T=1 << 20), b"too many"),
                     (dict(q_out=ctypes.c_void_p(4096 + 256), ldq=512), b"apart"),
                     (dict(q_out=P, ldq=512, T=2), b"apart")):
        kw.setdefault("kv", ref)
        assert fn(*rotary_args(**kw)) == -1, kw
        assert word in lib.fs_last_error(), (kw, lib.fs_last_error())
    assert fn(*rotary_args(kv=None)) == -1 and b"descriptor" in lib.fs_last_error()
    for kw in (dict(k=0), dict(table=0), dict(block_size=0), dict(num_blocks=0), dict(table_cols=0)):
        bad = quant_desc(**kw)
        assert fn(*rotary_args(kv=ctypes.byref(bad if quant else bad.cache))) == -1
    if quant:
        bad = quant_desc()
        bad.k_scale = None
        assert fn(*rotary_args(kv=ctypes.byref(bad))) == -1 and b"scales" in lib.fs_last_error()
    assert fn(*rotary_args(kv=None, B=0)) == 0


def test_dequant_and_decode_refusals(lib):
    d = quant_desc()
    ref = ctypes.byref(d)

    def deq(kv=ref, B=1, n=16, nkv=2, hd=128, k=P, v=P, dtype=L.FS_BF16):
        return lib.fs_kv_dequant(kv, B, n, nkv, hd, k, v, dtype, None)

    for kw, word in ((dict(kv=None), b"descriptor"), (dict(k=None), b"NULL"), (dict(dtype=5), b"dtype"),
                     (dict(hd=0), b"head"), (dict(nkv=0), b"head"), (dict(n=129), b"fewer slots"),
                     (dict(B=70000), b"too many"), (dict(n=1 << 40), b"too many")):
        assert deq(**kw) == -1 and word in lib.fs_last_error(), (kw, lib.fs_last_error())
    assert deq(n=0) == 0 and deq(B=0) == 0

    def dec(q=P, ldq=512, kv=ref, n=128, pos=P, out=P, ldo=512, B=1, nh=4, nkv=2, hd=128, ws=None, wsb=0,
            dtype=L.FS_BF16):
        return lib.fs_attention_decode_quant(q, ldq, kv, n, pos, out, ldo, B, nh, nkv, hd, 0.1, ws, wsb, dtype, None)

    for kw, word in ((dict(q=None), b"NULL"), (dict(out=None), b"NULL"), (dict(kv=None), b"descriptor"),
                     (dict(n=0), b"no slots"), (dict(n=129), b"fewer slots"), (dict(hd=258, ldq=4096, ldo=4096), b"head_dim"),
                     (dict(hd=63), b"head_dim"), (dict(nh=5), b"multiple"), (dict(nkv=0), b"multiple"),
                     (dict(nh=0), b"multiple"), (dict(ldq=500), b"stride"), (dict(ldo=500), b"stride"),
                     (dict(dtype=9), b"dtype"), (dict(B=70000), b"too many")):
        assert dec(**kw) == -1 and word in lib.fs_last_error(), (kw, lib.fs_last_error())
    long = quant_desc(table_cols=64, table_stride=64)
    need = lib.fs_attention_decode_quant_workspace(1, 4, 2, 128, 1024)
    assert need == 4 * 2 * 130 * 4 and lib.fs_attention_decode_quant_workspace(1, 4, 2, 128, 512) == 0
    for kw in (dict(), dict(ws=P, wsb=need - 1), dict(ws=ctypes.c_void_p(4097), wsb=need)):
        assert dec(kv=ctypes.byref(long), n=1024, **kw) == -1 and b"workspace" in lib.fs_last_error()
    assert dec(B=0) == 0


def test_descriptor_takes_strides_of_single_entries_as_they_come():
    """A dimension of one entry has no stride that matters: slices that differ there alone are one pool."""
    k = torch.zeros(4, 2, 8, 16).to(F8)
    s, t = torch.zeros(4, 2, 8), torch.zeros(1, 2, dtype=torch.int64)
    # one KV head, one slot a block, one block; v and the scales with memory of their own
    for cut in ((slice(None), slice(1, 2)), (slice(None), slice(None), slice(0, 1)), (slice(3, 4),),
                (slice(0, 1), slice(0, 1)), (slice(0, 1), slice(0, 1), slice(5, 6))):
        kc, sc = k[cut], s[cut]
        d = ops.quant_paged_desc(kc, kc.clone(memory_format=torch.contiguous_format), sc, sc.contiguous(), t) \
            if kc.shape[0] == 1 else ops.quant_paged_desc(kc, kc, sc, sc, t)
        assert d.cache.k == kc.data_ptr() and d.k_scale == sc.data_ptr()
        assert (d.cache.block_size, d.cache.num_blocks) == (kc.shape[2], kc.shape[0])
        assert d.cache.block_stride >= 0 and d.cache.block_stride % 16 == 0 and d.cache.head_stride % 16 == 0
    spread = s[:, :, ::8]                                            # one slot a block, slots eight apart
    assert spread.stride(2) == 8
    d = ops.quant_paged_desc(k[:, :, :1], k[:, :, :1], spread, spread, t)
    assert (d.scale_block_stride, d.scale_head_stride) == (16, 8)
    d = ops.quant_paged_desc(k[:, :1], k[:, :1], s[:, :1], s[:, :1], t)
    assert d.cache.block_stride == 256 and d.scale_block_stride == 16
    for args in ((k, torch.zeros(4, 4, 8, 16).to(F8)[:, :2], s, s, t), (k, k, s, torch.zeros(4, 4, 8)[:, :2], t)):
        with pytest.raises(ValueError, match="alike"):               # more than one entry: the strides have to agree
            ops.quant_paged_desc(*args)


@pytest.mark.parametrize("bad", [dict(factor=math.inf), dict(factor=math.nan), dict(factor="8"), dict(factor=None),
                                 dict(factor=[2.0]), dict(original_max_len=math.inf), dict(original_max_len="64"),
                                 dict(beta_fast=math.inf), dict(beta_fast=math.nan), dict(beta_slow="1"),
                                 dict(attn_factor=math.inf), dict(attn_factor=math.nan), dict(attn_factor=None)])
def test_config_refuses_rotary_numbers_that_are_none(bad):
    """Anything but finite numbers in rope_scaling is a ValueError when the model is described, not tables of zeros or
    NaN, or a TypeError, later."""
    scaling = {"kind": "by_parts", "factor": 2, "original_max_len": 64}
    ModelConfig(rope_scaling=scaling)
    with pytest.raises(ValueError, match="rope_scaling"):
        ModelConfig(rope_scaling={**scaling, **bad})
    with pytest.raises(ValueError, match="kind"):
        ModelConfig(rope_scaling={"kind": ["linear"], "factor": 2})
    if "factor" in bad:
        for kind in ("linear", "ntk"):
            with pytest.raises(ValueError, match="rope_scaling"):
                ModelConfig(rope_scaling={"kind": kind, **bad})


def test_config_refuses_rotary_dims_that_are_no_whole_numbers():
    for bad in (8.0, "8", True):
        with pytest.raises(ValueError, match="rotary_dim"):
            ModelConfig(rotary_dim=bad)


def test_dequant_for_queries_refusals(lib):
    d = quant_desc()

    def deq(kv=ctypes.byref(d), B=1, n=16, pos=P, T=3, k=P, v=P, dtype=L.FS_BF16):
        return lib.fs_kv_dequant_for(kv, B, n, 2, 128, pos, T, k, v, dtype, None)

    for kw, word in ((dict(pos=None), b"positions"), (dict(T=0), b"positions"), (dict(T=-1), b"positions"),
                     (dict(T=1 << 31), b"positions"), (dict(kv=None), b"descriptor"), (dict(v=None), b"NULL"),
                     (dict(dtype=5), b"dtype"), (dict(n=129), b"fewer slots"), (dict(B=70000), b"too many")):
        assert deq(**kw) == -1 and word in lib.fs_last_error(), (kw, lib.fs_last_error())
    assert deq(n=0, pos=None) == 0 and deq(B=0, T=0) == 0
