"""The general rotary write, the 8-bit cache's write and read-back, and decode attention over it, each against a plain
statement in 64 bits. Tolerances count roundings: half a step of the type a value is held in (bf16 2^-8, e4m3 2^-4 or
2^-10 below its normal range, f16 2^-11), and 2^-24 for each fp32 operation."""

import math
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from forgeserve_b200 import _lib as L
from forgeserve_b200 import Engine, ForgeModel, ModelConfig, PagedKVPool, generate, ops
from forgeserve_b200.model import _rope_write, layer_forward_, rope_tables
from oracle import forge_oracle as O

DEV = "cuda"
F8 = torch.float8_e4m3fn
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(autouse=True)
def _clean_device_errors():
    if torch.cuda.is_available():
        L.device_error(clear=True)
    yield
    if torch.cuda.is_available():
        assert L.device_error(clear=True) == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def quant_pool(nblk, nkv, bs, hd, seed):
    g = gen(seed)
    k, v = ((torch.randn(nblk, nkv, bs, hd, generator=g, device=DEV) * 130).clamp(-448, 448).to(F8) for _ in range(2))
    ks, vs = (torch.exp(torch.randn(nblk, nkv, bs, generator=g, device=DEV) * 0.4) * 0.0075 for _ in range(2))
    return k, v, ks, vs


def bits(t):
    return t.contiguous().view(torch.uint8)


# ------------------------------------------------------------------------------------------- rotary write

def rotate64(x, cos, sin, layout):
    """x (n, heads, hd) in 64 bits -> (rotated, sum of the magnitudes that each value was summed from)."""
    r = 2 * cos.shape[1]
    y, mag = x.clone(), x.abs()
    for i in range(r // 2):
        ia, ib = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
        c, s = cos[:, None, i], sin[:, None, i]
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


WRITE_CASES = [  # dtype, layout, B, T, nh, nkv, hd, rd, bs
    (torch.bfloat16, "half", 2, 5, 8, 2, 128, 128, 16),
    (torch.bfloat16, "interleaved", 2, 5, 8, 2, 128, 64, 16),
    (torch.bfloat16, "half", 1, 1, 32, 8, 128, 32, 16),
    (torch.bfloat16, "interleaved", 3, 33, 5, 5, 64, 64, 8),
    (torch.bfloat16, "half", 3, 7, 4, 1, 256, 64, 64),
    (torch.bfloat16, "half", 2, 9, 6, 3, 80, 20, 7),
    (torch.bfloat16, "interleaved", 2, 9, 6, 3, 80, 78, 1),
    (torch.bfloat16, "half", 2, 9, 6, 3, 96, 96, 16),
    (torch.bfloat16, "interleaved", 1, 3, 1, 1, 2, 2, 3),
    (torch.bfloat16, "half", 1, 17, 3, 1, 512, 512, 5),
    (torch.float32, "half", 2, 19, 8, 4, 64, 64, 16),
    (torch.float32, "interleaved", 2, 3, 7, 7, 128, 126, 16),
    (torch.float32, "half", 4, 2, 3, 1, 32, 16, 4),
    (torch.float32, "interleaved", 1, 40, 2, 2, 112, 30, 20),
    (torch.float32, "half", 1, 5, 3, 3, 18, 6, 2),
    (torch.bfloat16, "half", 2, 600, 32, 8, 128, 128, 16),
    # heads whose lanes are no power of two: some hold nothing
    (torch.bfloat16, "interleaved", 3, 50, 6, 3, 96, 96, 16),
    (torch.bfloat16, "interleaved", 3, 50, 6, 3, 48, 24, 16),
    (torch.bfloat16, "half", 3, 50, 5, 5, 112, 64, 16),
    (torch.float32, "interleaved", 3, 50, 6, 3, 80, 80, 16),
    (torch.float32, "half", 3, 50, 7, 1, 176, 176, 16),
    # halves that are no whole pieces
    (torch.bfloat16, "half", 3, 50, 8, 2, 128, 126, 16),
    (torch.bfloat16, "half", 3, 50, 6, 3, 80, 40, 8),
    (torch.bfloat16, "half", 2, 33, 5, 1, 512, 2, 16),
    (torch.bfloat16, "half", 5, 20, 7, 7, 16, 14, 4),
    (torch.float32, "half", 3, 50, 5, 5, 32, 30, 16),
    (torch.float32, "half", 2, 21, 3, 1, 256, 254, 16),
    (torch.float32, "half", 2, 21, 6, 2, 112, 12, 20),
    (torch.bfloat16, "half", 2, 600, 32, 8, 128, 100, 16),
    # more items than a wave of CTAs takes at once
    (torch.bfloat16, "half", 3, 1500, 5, 2, 64, 64, 16),
    (torch.bfloat16, "half", 2, 3000, 40, 8, 16, 16, 16),
    (torch.bfloat16, "interleaved", 2, 900, 16, 8, 128, 128, 16),
    (torch.bfloat16, "interleaved", 1, 9000, 1, 1, 128, 64, 32),
    (torch.float32, "interleaved", 2, 700, 9, 3, 80, 80, 7),
    (torch.float32, "half", 3, 500, 32, 8, 128, 128, 16),
    (torch.float32, "half", 2, 800, 11, 1, 64, 62, 16),
    (torch.bfloat16, "half", 3, 700, 12, 4, 208, 208, 16),
    (torch.bfloat16, "half", 3, 700, 12, 4, 272, 270, 16),
    (torch.float32, "interleaved", 3, 700, 6, 2, 24, 24, 16),
    # past 128 MiB of rows
    (torch.bfloat16, "half", 3, 3500, 40, 8, 128, 128, 64),
    (torch.float32, "interleaved", 1, 4700, 40, 9, 128, 64, 64),
]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("case", WRITE_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotary_write(case, quant):
    dtype, layout, B, T, nh, nkv, hd, rd, bs = case
    g = gen(1)
    starts = [11 * i for i in range(B)]
    S = max(starts) + T
    cols = -(-S // bs)
    table = torch.randperm(B * cols + 2, generator=g, device=DEV)[: B * cols].view(B, cols)
    pos = torch.tensor(starts, device=DEV)[:, None] + torch.arange(T, device=DEV)
    if T > 2:
        pos[-1, T - T // 3 - 1:] = -1                               # a padded row
    cos, sin = (t.to(DEV) for t in rope_tables(rd, S, 10000.0))
    qkv = torch.randn(B * T, (nh + 2 * nkv) * hd, generator=g, device=DEV).mul_(
        torch.exp(torch.randn((nh + 2 * nkv) * hd, generator=g, device=DEV))).to(dtype)
    qkv0 = qkv.clone()
    shape = (B * cols + 2, nkv, bs, hd)
    if quant:
        pools = quant_pool(*shape, seed=2)
        desc = ops.quant_paged_desc(*pools, table)
    else:
        pools = tuple(torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
        desc = ops.paged_desc(*pools, table)
    before = [p.clone() for p in pools]
    q_out = torch.full((B * T, nh * hd), 7.0, dtype=dtype, device=DEV)
    ops.rotary_kv_write(qkv, cos, sin, pos, desc, B, T, nh, nkv, hd, layout=layout, q_out=q_out)
    assert torch.equal(qkv, qkv0)

    row, col = torch.nonzero(pos >= 0, as_tuple=True)
    p = pos[row, col]
    x = qkv0.view(B, T, nh + 2 * nkv, hd)[row, col].double()
    y, mag = rotate64(x[:, : nh + nkv], cos.double()[p], sin.double()[p], layout)
    err = 3 * U * mag                                               # two products and their sum
    q_got = q_out.view(B, T, nh, hd)
    assert (q_got[pos < 0] == 7.0).all()                            # padding: left as it was
    diff = (q_got[row, col].double() - y[:, :nh]).abs()
    assert (diff <= HALF[dtype] * y[:, :nh].abs() + 2 * err[:, :nh]).all()
    block, slot = table[row, p // bs], p % bs
    written = torch.zeros(shape[:3], dtype=torch.bool, device=DEV)
    written[block, :, slot] = True
    for i, (want, e) in enumerate([(y[:, nh:], err[:, nh:]), (x[:, nh + nkv:], torch.zeros_like(x[:, nh + nkv:]))]):
        got = pools[i][block, :, slot] if not quant else bits(pools[i]).view(shape)[block, :, slot].view(F8)
        assert torch.equal(bits(pools[i]).view(*shape[:3], -1)[~written], bits(before[i]).view(*shape[:3], -1)[~written])
        if not quant:
            assert ((got.double() - want).abs() <= HALF[dtype] * want.abs() + 2 * e).all()
            continue
        top = want.abs().amax(-1)
        scale = (top / 448).clamp_min(2.0 ** -126)
        s_got = pools[2 + i][block, :, slot].double()
        s_err = (e.amax(-1) / 448) + 2 * U * scale                  # the largest value's error, the division
        assert ((s_got - scale).abs() <= s_err).all()
        assert torch.equal(pools[2 + i][~written], before[2 + i][~written])
        # the code is x / scale to half a step; its argument carries the errors of x and of 1 / scale
        z = want / scale[..., None]
        arg = (e + z.abs() * s_err[..., None]) / scale[..., None] + 4 * U * z.abs()
        step = torch.maximum(z.abs() * 2.0 ** -4, torch.full_like(z, 2.0 ** -10))
        assert ((got.double() - z).abs() <= step * (1 + 2.0 ** -20) + 2 * arg).all()
    # in place: the same values in q's place, k and v of qkv untouched
    ops.rotary_kv_write(qkv, cos, sin, pos, desc, B, T, nh, nkv, hd, layout=layout)
    real = (pos >= 0).view(-1)
    assert torch.equal(qkv[real, : nh * hd], q_out[real])
    assert torch.equal(qkv[~real], qkv0[~real]) and torch.equal(qkv[:, nh * hd:], qkv0[:, nh * hd:])


def test_rotary_write_contiguous_cache_and_strided_rows():
    """A per-row cache (slots appended at slot_base), qkv rows that are slices of a wider tensor, rows of q_out apart."""
    B, T, nh, nkv, hd, base, cap = 2, 6, 4, 2, 64, 5, 16
    for dtype in (torch.bfloat16, torch.float32):
        for off in (0, 3):                                          # 3: rows off the vector alignment
            wide = torch.randn(B * T, (nh + 2 * nkv) * hd + 19, generator=gen(3), device=DEV).to(dtype)
            qkv = wide[:, off: off + (nh + 2 * nkv) * hd]
            k = torch.zeros(B, nkv, cap, hd, dtype=dtype, device=DEV)
            v = torch.zeros_like(k)
            pos = (base + torch.arange(T, device=DEV)).expand(B, T).contiguous()
            cos, sin = (t.to(DEV) for t in rope_tables(32, 64, 10000.0))
            q = torch.zeros(B * T, nh * hd + 5, dtype=dtype, device=DEV)[:, : nh * hd]
            from forgeserve_b200.kv import row_table
            ops.rotary_kv_write(qkv, cos, sin, pos, ops.contiguous_desc(k, v, row_table(B, torch.device(DEV))), B, T,
                                nh, nkv, hd, slot_base=base, slot_from_pos=False, layout="interleaved", q_out=q)
            x = qkv.reshape(B * T, nh + 2 * nkv, hd).double()
            y, mag = rotate64(x[:, : nh + nkv], cos.double()[pos.view(-1)], sin.double()[pos.view(-1)], "interleaved")
            tol = HALF[dtype] * y.abs() + 6 * U * mag
            assert ((q.reshape(B * T, nh, hd).double() - y[:, :nh]).abs() <= tol[:, :nh]).all()
            got = k[:, :, base: base + T].transpose(1, 2).reshape(B * T, nkv, hd).double()
            assert ((got - y[:, nh:]).abs() <= tol[:, nh:]).all()
            assert torch.equal(v[:, :, base: base + T].transpose(1, 2).reshape(B * T, nkv, hd).double(), x[:, nh + nkv:])
            assert not k[:, :, :base].any() and not k[:, :, base + T:].any()


@pytest.mark.parametrize("hd", [128, 80, 18])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_store_special_rows(dtype, hd):
    """Rows of zeros, of the smallest and largest values, with an infinity, with a NaN; each alone in its row."""
    rows = torch.zeros(8, hd, device=DEV)
    rows[1] = 1e-44 if dtype == torch.float32 else 1e-40
    rows[2, 3] = -2.0 ** -120
    rows[3] = 3.0e38
    rows[4], rows[4, 5] = 1.0, math.inf
    rows[5], rows[5, 7] = 1.0, math.nan
    rows[6], rows[6, 1] = 1.0, -math.inf
    rows[7] = torch.linspace(-448, 448, hd, device=DEV)
    x = rows.to(dtype)
    T = 8
    k, v, ks, vs = quant_pool(1, 1, 8, hd, 1)
    qkv = torch.cat([x, x.flip(0)], 1)                               # nh = 0: k and v only
    table = torch.zeros(1, 1, dtype=torch.int64, device=DEV)
    desc = ops.quant_paged_desc(k, v, ks, vs, table)
    ops.rotary_kv_write(qkv, None, None, torch.arange(T, device=DEV), desc, 1, T, 0, 1, hd)
    for codes, scale, src in ((k, ks, x), (v, vs, x.flip(0))):
        codes, scale, src = codes[0, 0].double(), scale[0, 0].double(), src.double()
        got = codes * scale[:, None]
        ok = torch.isfinite(src).all(-1)
        assert torch.isnan(got[~ok]).all()
        top = src.abs().amax(-1)
        want_scale = (top / 448).clamp_min(2.0 ** -126)
        assert ((scale - want_scale).abs()[ok] <= 2 * U * want_scale[ok]).all()
        tol = torch.maximum(src.abs() * 2.0 ** -4, want_scale[:, None] * 2.0 ** -10) * (1 + 2.0 ** -18)
        assert ((got - src).abs() <= tol)[ok].all()
    kd, vd = ops.kv_dequant(desc, 1, 8, 1, hd, torch.float32)
    assert torch.equal(torch.isnan(kd[0, 0]).any(-1), ~torch.isfinite(x).all(-1))
    assert torch.equal(torch.isnan(vd[0, 0]).any(-1), ~torch.isfinite(x.flip(0)).all(-1))


@pytest.mark.parametrize("hd,rd", [(128, 128), (128, 64), (80, 20)])
@pytest.mark.parametrize("quant", [False, True])
def test_write_bad_positions_and_slots_are_flagged_and_skipped(quant, hd, rd):
    nh, nkv, bs = 4, 2, 4
    cos, sin = (t.to(DEV) for t in rope_tables(rd, 32, 10000.0))
    qkv = torch.randn(5, (nh + 2 * nkv) * hd, generator=gen(5), device=DEV).bfloat16()
    pools = quant_pool(6, nkv, bs, hd, 3) if quant else tuple(torch.zeros(6, nkv, bs, hd, device=DEV).bfloat16()
                                                              for _ in range(2))
    table = torch.tensor([[1, 99, -3, 2]], device=DEV)
    desc = (ops.quant_paged_desc if quant else ops.paged_desc)(*pools, table)
    before = [p.clone() for p in pools]
    q = torch.zeros(5, nh * hd, device=DEV).bfloat16()
    # in the tables and the cache; block 99; block -3; past the block table; past the rotation tables
    ops.rotary_kv_write(qkv, cos, sin, torch.tensor([0, 5, 9, 20, 40], device=DEV), desc, 1, 5, nh, nkv, hd, q_out=q)
    assert L.device_error(clear=True) == L.FS_ERR_BAD_SLOT | L.FS_ERR_BAD_POSITION
    assert q[:4].any(-1).all() and not q[4].any()
    for now, was in zip(pools, before):
        changed = (bits(now) != bits(was)).view(*now.shape[:3], -1).any(-1)
        assert changed.sum() == nkv and changed[1, :, 0].all()      # token 0 alone was stored


# ------------------------------------------------------------------------------------------------ read-back

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,slots,nkv,hd,bs", [(1, 1, 1, 128, 16), (2, 37, 3, 128, 16), (3, 100, 2, 64, 7),
                                               (1, 515, 1, 80, 1), (2, 33, 2, 18, 16), (2, 5, 1, 256, 64),
                                               (1, 70, 2, 6, 16), (2, 300, 8, 128, 300)])
def test_dequant_is_the_rounded_product(dtype, B, slots, nkv, hd, bs):
    cols = -(-slots // bs)
    k, v, ks, vs = quant_pool(B * cols + 3, nkv, bs, hd, 7)
    table = torch.randperm(B * cols + 3, generator=gen(8), device=DEV)[: B * cols].view(B, cols)
    kd, vd = ops.kv_dequant(ops.quant_paged_desc(k, v, ks, vs, table), B, slots, nkv, hd, dtype)
    for got, c, s in ((kd, k, ks), (vd, v, vs)):
        want = (bits(c).view(c.shape)[table].view(F8).float() * s[table][..., None]).transpose(1, 2).reshape(
            B, nkv, cols * bs, hd)[:, :, :slots].to(dtype)
        assert torch.equal(got, want)


def test_dequant_bad_block_reads_zeros_and_no_slots_is_empty():
    k, v, ks, vs = quant_pool(4, 2, 4, 64, 9)
    desc = ops.quant_paged_desc(k, v, ks, vs, torch.tensor([[1, 4, -1, 2]], device=DEV))
    kd, vd = ops.kv_dequant(desc, 1, 15, 2, 64, torch.bfloat16)
    assert L.device_error(clear=True) == L.FS_ERR_BAD_SLOT
    assert not kd[:, :, 4:12].any() and not vd[:, :, 4:12].any()
    assert kd[:, :, :4].any() and kd[:, :, 12:].any()
    kd, vd = ops.kv_dequant(desc, 1, 0, 2, 64, torch.bfloat16)
    assert kd.shape == (1, 2, 0, 64)


# ------------------------------------------------------------------------------------------ decode attention

def decode_ref(q, k, v, ks, vs, table, positions, n_slots, nh, nkv, hd):
    """(out, bound on its error before the last rounding) in 64 bits, row by row."""
    B, bs, rep = q.shape[0], k.shape[2], nh // nkv
    out = torch.zeros(B, nh * hd, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    half_p = 2.0 ** -11 + 2.0 ** -12 if q.dtype == torch.bfloat16 else 2.0 ** -21
    for r in range(B):
        n = min(int(positions[r]) + 1, n_slots)
        if n <= 0:
            continue
        t = torch.arange(n, device=DEV)
        blk, s = table[r][t // bs], t % bs
        kk, vv = (c.view(torch.uint8)[blk, :, s].view(F8).double().transpose(0, 1) for c in (k, v))   # nkv, n, hd
        ksr, vsr = ks[blk, :, s].double().t(), vs[blk, :, s].double().t()
        qq = q[r].double().view(nkv, rep, hd)
        score = torch.einsum("grd,gnd->grn", qq, kk) * ksr[:, None] / math.sqrt(hd)
        p = torch.softmax(score, -1)
        vd = vv * vsr[..., None]
        out[r] = torch.einsum("grn,gnd->grd", p, vd).reshape(-1)
        # a score is off by hd + 8 fp32 roundings of its magnitudes (q held to 2^-25 of its largest value at worst), a
        # probability by that much relative to itself and by the type that it enters the product in
        mag = torch.einsum("grd,gnd->grn", qq.abs(), kk.abs()) * ksr.abs()[:, None] / math.sqrt(hd)
        ds = ((hd + 8) * U * mag).amax(-1)
        qerr = qq.abs().amax(-1) * (2.0 ** -25) * (kk.abs().sum(-1) * ksr.abs()).amax(-1)[:, None] / math.sqrt(hd)
        rel = 2 * (ds + (qerr if q.dtype == torch.bfloat16 else 0)) + half_p + (n + 64) * U
        absum = torch.einsum("grn,gnd->grd", p, vd.abs())
        # probabilities below the f16 range are off by 2^-25 of the largest p vs at most
        floor = (p * vsr.abs()[:, None]).amax(-1) * 2.0 ** -24 * vv.abs().sum(1).amax(-1)[:, None]
        bound[r] = (absum * rel[..., None] + floor[..., None]).reshape(-1)
    return out, bound


def decode_case(dtype, lengths, nh, nkv, hd, bs, seed=1, spare_cols=0):
    B = len(lengths)
    cols = max(1, -(-max(lengths) // bs)) + spare_cols
    nblk = B * cols + 3
    pools = quant_pool(nblk, nkv, bs, hd, seed)
    table = torch.randperm(nblk, generator=gen(seed), device=DEV)[: B * cols].view(B, cols)
    positions = torch.tensor(lengths, device=DEV) - 1
    q = (torch.randn(B, nh * hd, generator=gen(seed + 1), device=DEV) * 1.5).to(dtype)
    return q, pools, table, positions, cols * bs


def check_decode(q, pools, table, positions, n_slots, nh, nkv, hd):
    out = torch.full_like(q, 9.0)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n_slots, positions, out, q.shape[0], nh, nkv, hd)
    want, bound = decode_ref(q, *pools, table, positions, n_slots, nh, nkv, hd)
    # below 2^-126 a type's steps no longer shrink: bf16 (7 fraction bits) has steps of 2^-133, half of one is 2^-134;
    # fp32 sums of such values round at 2^-150 each
    tiny = 2.0 ** -134 if q.dtype == torch.bfloat16 else n_slots * 2.0 ** -150
    tol = HALF[q.dtype] * (want.abs() + bound) + bound + tiny
    worst = ((out.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst
    return out


DECODE_CASES = [  # dtype, lengths, nh, nkv, hd, bs
    (torch.bfloat16, [1], 32, 8, 128, 16),
    (torch.bfloat16, [16, 17, 15, 1, 0], 32, 8, 128, 16),
    (torch.bfloat16, [512, 513, 511, 1024, 0], 8, 2, 128, 16),
    (torch.bfloat16, [1300, 77], 64, 8, 128, 64),
    (torch.bfloat16, [700, 33], 16, 1, 128, 32),
    (torch.bfloat16, [700, 33], 24, 1, 64, 16),
    (torch.bfloat16, [90, 600], 12, 4, 64, 16),
    (torch.bfloat16, [90, 600], 7, 7, 64, 8),
    (torch.bfloat16, [41, 530], 8, 4, 256, 16),
    (torch.bfloat16, [41, 530], 14, 2, 256, 5),
    (torch.bfloat16, [100, 523], 10, 2, 128, 20),
    (torch.bfloat16, [100, 523], 10, 2, 128, 1),
    (torch.bfloat16, [100, 523], 4, 2, 80, 16),
    (torch.bfloat16, [100, 523], 4, 2, 32, 16),
    (torch.bfloat16, [64], 6, 2, 18, 3),
    (torch.bfloat16, [9000], 32, 8, 128, 16),
    (torch.bfloat16, [700], 8, 2, 128, 700),
    (torch.float32, [1, 0, 17], 8, 4, 128, 16),
    (torch.float32, [1200, 513, 512], 8, 2, 128, 16),
    (torch.float32, [640, 30], 12, 12, 64, 20),
    (torch.float32, [640, 30], 32, 2, 64, 16),
    (torch.float32, [640, 30], 9, 1, 256, 48),
    (torch.float32, [640, 30], 4, 2, 96, 16),
    (torch.float32, [70], 3, 3, 6, 2),
    # head sizes between the ones that the tensor-core kernel is built for
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 16, 16),
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 48, 10),
    (torch.bfloat16, [100, 523, 31, 0], 18, 2, 96, 32),
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 112, 16),
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 144, 16),
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 192, 9),
    (torch.bfloat16, [100, 523, 31, 0], 20, 2, 240, 16),
    (torch.float32, [100, 523, 31, 0], 8, 2, 80, 16),
    (torch.float32, [100, 523, 31, 0], 20, 2, 208, 16),
    (torch.float32, [100, 523, 31, 0], 8, 2, 32, 3),
    (torch.bfloat16, [100, 523, 31, 0], 8, 2, 40, 16),
    # rows long enough for splits of several units of 512 slots, beside short ones
    (torch.bfloat16, [19000, 700, 9500, 4700], 64, 64, 64, 16),
    (torch.bfloat16, [11000, 513, 5000], 256, 128, 128, 24),
    (torch.float32, [6000, 40], 200, 200, 64, 16),
    (torch.bfloat16, [6000, 3100], 100, 100, 32, 16),
]


@pytest.mark.parametrize("case", DECODE_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_decode(case):
    dtype, lengths, nh, nkv, hd, bs = case
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs)
    out = check_decode(q, pools, table, positions, n_slots, nh, nkv, hd)
    for r, n in enumerate(lengths):
        if n == 0:
            assert not out[r].any()


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(torch.bfloat16, 8, 2, 128), (torch.float32, 8, 2, 128),
                                             (torch.bfloat16, 4, 2, 80), (torch.bfloat16, 4, 2, 40),
                                             (torch.float32, 4, 1, 256)])
def test_decode_does_not_read_past_the_visible_slots(dtype, nh, nkv, hd):
    """NaN scales and codes behind each row's last slot, in unused blocks and past n_slots change nothing."""
    lengths = [1, 15, 530, 517]
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, 16, spare_cols=2)
    clean = check_decode(q, pools, table, positions, n_slots, nh, nkv, hd)
    seen = torch.zeros(pools[0].shape[:3], dtype=torch.bool, device=DEV)
    for r, n in enumerate(lengths):
        t = torch.arange(n, device=DEV)
        seen[table[r][t // 16], :, t % 16] = True
    pools[2][~seen] = math.nan
    pools[3][~seen] = math.inf
    for p in pools[:2]:
        p.view(torch.uint8)[~seen] = 0x7F
    assert torch.equal(check_decode(q, pools, table, positions, n_slots, nh, nkv, hd), clean)
    # positions past n_slots see n_slots slots
    out = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), 1, positions + 10, out, 4, nh, nkv, hd)
    first, _ = decode_ref(q, *pools, table, torch.zeros_like(positions), 1, nh, nkv, hd)
    assert ((out.double() - first).abs() <= (HALF[dtype] + 2.0 ** -9) * first.abs() + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [128, 80, 40])
def test_decode_special_values(dtype, hd):
    """NaN and infinity in a visible key or value reach their row and KV head only; rows of zero scale, queries far out
    of the half range, values whose scales span many powers of two."""
    nh, nkv, bs = 4, 2, 16
    lengths = [600, 600, 600, 600, 600, 600]
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs, seed=5)
    k, v, ks, vs = pools

    def at(r, slot):
        return table[r, slot // bs], slot % bs

    b, s = at(0, 523)
    ks[b, 0, s] = math.nan
    b, s = at(1, 10)
    vs[b, 1, s] = math.inf
    b, s = at(2, 599)
    v.view(torch.uint8)[b, 1, s, 3] = 0x7F
    out = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n_slots, positions, out, 6, nh, nkv, hd)
    o = out.view(6, nkv, nh // nkv, hd)
    assert torch.isnan(o[0, 0]).all() and torch.isfinite(o[0, 1]).all()
    assert not torch.isfinite(o[1, 1]).any() and torch.isfinite(o[1, 0]).all()   # code * infinity
    assert torch.isnan(o[2, 1, :, 3]).all() and torch.isfinite(o[2, 1, :, :3]).all() and torch.isfinite(o[2, 0]).all()
    assert torch.isfinite(o[3:]).all()
    # values: zero scales, scales from 2^-60 to 2^60; queries of 1e30 against keys of 1e-30
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs, seed=6)
    k, v, ks, vs = pools
    vs[table[0]] = 0.0
    vs[table[1]] *= torch.exp2(torch.randint(-60, 60, vs[table[1]].shape, generator=gen(4), device=DEV).float())
    ks[table[2]] *= 1e-30
    q[2] = (q[2].double() * 1e30).to(dtype)
    ks[table[3]] *= 30.0                                            # scores of several hundred: one key takes it all
    vs[table[3]] *= 2.0 ** 123                                      # values near fp32's end
    v.view(torch.uint8)[table[3]] &= 0x8F                           # (their codes below 0.02, so that none leaves it)
    vs[table[4]] *= 1e-38
    q[5] = 0.0
    out = check_decode(q, pools, table, positions, n_slots, nh, nkv, hd)
    assert not out[0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [128, 40])
def test_decode_nan_and_infinity_in_a_query_stay_in_their_head(dtype, hd):
    q, pools, table, positions, n_slots = decode_case(dtype, [600, 40, 9], 8, 2, hd, 16)
    want, bound = (x.view(3, 8, hd) for x in decode_ref(q, *pools, table, positions, n_slots, 8, 2, hd))
    bad = q.clone().view(3, 8, hd)
    bad[0, 1, 3], bad[1, 6, 0], bad[2, 4, hd - 1] = math.nan, math.inf, -math.inf
    out = torch.empty_like(q)
    ops.attention_decode_quant(bad.view(3, -1), ops.quant_paged_desc(*pools, table), n_slots, positions, out, 3, 8, 2, hd)
    out = out.double().view(3, 8, hd)
    hit = torch.zeros(3, 8, dtype=torch.bool, device=DEV)
    hit[0, 1] = hit[1, 6] = hit[2, 4] = True
    assert torch.isnan(out[hit]).all()
    tol = HALF[dtype] * (want.abs() + bound) + bound
    assert ((out - want).abs() <= tol)[~hit].all()


def test_decode_bad_block_is_flagged_and_reads_zero():
    for dtype, hd in ((torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 48)):
        q, pools, table, positions, n_slots = decode_case(dtype, [40, 64], 4, 2, hd, 16)
        good = table.clone()
        table[0, 1], table[1, 3] = 1 << 40, -1
        out = torch.empty_like(q)
        ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n_slots, positions, out, 2, 4, 2, hd)
        assert L.device_error(clear=True) == L.FS_ERR_BAD_SLOT
        zero = [torch.cat([p, torch.zeros_like(p[:1].float()).to(p.dtype)]) for p in pools]
        good[0, 1] = good[1, 3] = zero[0].shape[0] - 1
        want, bound = decode_ref(q, *zero, good, positions, n_slots, 4, 2, hd)
        assert ((out.double() - want).abs() <= HALF[dtype] * (want.abs() + bound) + bound).all()


def test_decode_offsets_past_32_bits():
    """A pool whose codes pass 4 GiB: the rows at its end are read and written where they lie."""
    nkv, bs, hd, nh = 8, 256, 128, 16
    nblk = (1 << 32) // (nkv * bs * hd) + 40
    k = torch.zeros(nblk, nkv, bs, hd, dtype=torch.uint8, device=DEV).view(F8)
    v = torch.zeros_like(k.view(torch.uint8)).view(F8)
    ks, vs = (torch.zeros(nblk, nkv, bs, device=DEV) for _ in range(2))
    table = torch.tensor([[nblk - 1, nblk - 7, 3]], device=DEV)
    desc = ops.quant_paged_desc(k, v, ks, vs, table)
    T = 600
    pos = torch.arange(T, device=DEV)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, generator=gen(1), device=DEV).bfloat16()
    cos, sin = (t.to(DEV) for t in rope_tables(hd, T, 10000.0))
    q = torch.empty(T, nh * hd, dtype=torch.bfloat16, device=DEV)
    ops.rotary_kv_write(qkv, cos, sin, pos, desc, 1, T, nh, nkv, hd, q_out=q)
    small = [torch.zeros(3, *p.shape[1:], dtype=torch.uint8 if p.dtype == F8 else p.dtype, device=DEV) for p in (k, v, ks, vs)]
    small = [s.view(F8) if s.dtype == torch.uint8 else s for s in small]
    sdesc = ops.quant_paged_desc(*small, torch.tensor([[0, 1, 2]], device=DEV))
    ops.rotary_kv_write(qkv, cos, sin, pos, sdesc, 1, T, nh, nkv, hd, q_out=torch.empty_like(q))
    for big, sm in zip((k, v, ks, vs), small):
        for i, b in enumerate(table[0].tolist()):
            assert torch.equal(bits(big[b]), bits(sm[i]))
    outs = []
    for d in (desc, sdesc):
        out = torch.empty(1, nh * hd, dtype=torch.bfloat16, device=DEV)
        ops.attention_decode_quant(q[-1:], d, T, pos[-1:], out, 1, nh, nkv, hd)
        outs.append((out, *ops.kv_dequant(d, 1, T, nkv, hd, torch.bfloat16)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_decode_is_independent_of_batch_and_table_width():
    """The same row gives the same bits alone, in a batch, and behind a wider table."""
    nh, nkv, hd, bs = 16, 4, 128, 16
    q, pools, table, positions, n_slots = decode_case(torch.bfloat16, [1700, 60, 900], nh, nkv, hd, bs)
    whole = check_decode(q, pools, table, positions, n_slots, nh, nkv, hd)
    wide = torch.cat([table, torch.zeros_like(table)], 1)
    out = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, wide), 2 * n_slots, positions, out, 3, nh, nkv, hd)
    assert torch.equal(out, whole)
    for r in range(3):
        one = torch.empty_like(q[:1])
        ops.attention_decode_quant(q[r: r + 1], ops.quant_paged_desc(*pools, table[r: r + 1]), n_slots,
                                   positions[r: r + 1], one, 1, nh, nkv, hd)
        assert torch.equal(one[0], whole[r])


@pytest.mark.parametrize("dtype,nh,nkv,hd,bs", [(torch.bfloat16, 32, 4, 128, 16), (torch.float32, 32, 16, 64, 16),
                                                (torch.bfloat16, 32, 8, 128, 20), (torch.bfloat16, 32, 8, 40, 16),
                                                (torch.bfloat16, 128, 8, 128, 16)])
def test_decode_bits_do_not_depend_on_the_batch(dtype, nh, nkv, hd, bs):
    """Rows of a batch large enough for another join, and behind a table of other width, against each row alone."""
    lengths = [1 + (i * 797) % 3000 for i in range(40)]
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs, seed=11)
    whole = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n_slots, positions, whole, 40, nh, nkv, hd)
    wide = torch.cat([table] * 14, 1)
    out = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, wide), 14 * n_slots, positions, out, 40, nh, nkv, hd)
    assert torch.equal(out, whole)
    for r in (0, 7, 19, 39):
        one = torch.empty_like(q[:1])
        ops.attention_decode_quant(q[r: r + 1], ops.quant_paged_desc(*pools, table[r: r + 1]), n_slots,
                                   positions[r: r + 1], one, 1, nh, nkv, hd)
        assert torch.equal(one[0], whole[r])


@pytest.mark.parametrize("dtype,bs", [(torch.bfloat16, 16), (torch.bfloat16, 20), (torch.float32, 48)])
def test_decode_takes_several_splits_in_turn(dtype, bs):
    """A batch with more splits than CTAs are launched for: each row as it comes alone, one row against 64 bits."""
    nh, nkv, hd, B = 32, 32, 64, 48
    lengths = [1 + (i * 1237) % 5000 for i in range(B)]
    lengths[5] = 0
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs, seed=12)
    whole = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n_slots, positions, whole, B, nh, nkv, hd)
    assert not whole[5].any()
    for r in (0, 5, 11, 23, 47, max(range(B), key=lambda i: lengths[i])):
        one = torch.empty_like(q[:1])
        ops.attention_decode_quant(q[r: r + 1], ops.quant_paged_desc(*pools, table[r: r + 1]), n_slots,
                                   positions[r: r + 1], one, 1, nh, nkv, hd)
        assert torch.equal(one[0], whole[r])
    r = max(range(B), key=lambda i: lengths[i])
    check_decode(q[r: r + 1], pools, table[r: r + 1], positions[r: r + 1], n_slots, nh, nkv, hd)


def test_pool_slices_and_strided_rows():
    """Heads of a larger pool, rows of q and out inside wider tensors, a table cut from a wider one."""
    nkv, hd, bs, nh = 2, 128, 16, 8
    q0, pools, table, positions, n_slots = decode_case(torch.bfloat16, [600, 31], 3 * nh, 3 * nkv, hd, bs)
    cut = [p[:, 2:4] for p in pools]
    q = q0[:, hd * 3: hd * 3 + nh * hd]
    wide = torch.cat([table, table], 1)[:, : table.shape[1]]
    out = torch.zeros(2, nh * hd + 24, dtype=torch.bfloat16, device=DEV)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*cut, wide), n_slots, positions, out[:, 8: 8 + nh * hd], 2, nh,
                               nkv, hd)
    want, bound = decode_ref(q.contiguous(), *[c.contiguous() for c in cut], table, positions, n_slots, nh, nkv, hd)
    assert ((out[:, 8: 8 + nh * hd].double() - want).abs() <= 2.0 ** -8 * (want.abs() + bound) + bound).all()
    assert not out[:, :8].any() and not out[:, 8 + nh * hd:].any()
    kd, _ = ops.kv_dequant(ops.quant_paged_desc(*cut, wide), 2, 30, nkv, hd, torch.float32)
    full, _ = ops.kv_dequant(ops.quant_paged_desc(*pools, table), 2, 30, 3 * nkv, hd, torch.float32)
    assert torch.equal(kd, full[:, 2:4])


# ---------------------------------------------------------------------------------- streams, graphs, together

def chain(pools, table, qkv, cos, sin, positions, lengths_slots, nh, nkv, hd):
    """One decode step as a layer makes it: rotate and store the new token, attend, read back."""
    B = qkv.shape[0]
    desc = ops.quant_paged_desc(*pools, table)
    q = torch.empty(B, nh * hd, dtype=qkv.dtype, device=DEV)
    ops.rotary_kv_write(qkv, cos, sin, positions, desc, B, 1, nh, nkv, hd, q_out=q)
    out = ops.attention_decode_quant(q, desc, lengths_slots, positions, torch.empty_like(q), B, nh, nkv, hd)
    return out, ops.kv_dequant(desc, B, 20, nkv, hd, qkv.dtype)


def test_two_captured_graphs_and_another_stream():
    """Two graphs of the chain, captured one after another and replayed at once on two streams, give what eager calls on
    the default stream give, replay after replay."""
    nh, nkv, hd, bs = 16, 4, 128, 16
    cos, sin = (t.to(DEV) for t in rope_tables(hd, 4096, 10000.0))
    sets = []
    for seed in (1, 2):
        q, pools, table, positions, n_slots = decode_case(torch.bfloat16, [1500, 700], nh, nkv, hd, bs, seed=seed)
        qkv = torch.randn(2, (nh + 2 * nkv) * hd, generator=gen(seed), device=DEV).bfloat16()
        sets.append((pools, table, qkv, cos, sin, positions, n_slots, nh, nkv, hd))
    want = []
    for s in sets:
        out, (kd, vd) = chain(*s)
        want.append((out.clone(), kd.clone(), vd.clone()))
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, st in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs.append(chain(*s))
        graphs.append(g)
    for _ in range(20):
        for o, (kd, vd) in outs:
            o.fill_(3.0)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for (o, (kd, vd)), (wo, wk, wv) in zip(outs, want):
            assert torch.equal(o, wo) and torch.equal(kd, wk) and torch.equal(vd, wv)


def test_a_side_stream_and_two_threads():
    """The chain on a stream of its own, and from two host threads at once on two streams, gives the default stream's
    bits."""
    import threading

    nh, nkv, hd, bs = 8, 2, 64, 16
    cos, sin = (t.to(DEV) for t in rope_tables(hd, 4096, 10000.0))
    sets, want = [], []
    for seed in (3, 4):
        q, pools, table, positions, n_slots = decode_case(torch.bfloat16, [1500, 700], nh, nkv, hd, bs, seed=seed)
        qkv = torch.randn(2, (nh + 2 * nkv) * hd, generator=gen(seed), device=DEV).bfloat16()
        sets.append((pools, table, qkv, cos, sin, positions, n_slots, nh, nkv, hd))
        out, (kd, vd) = chain(*sets[-1])
        want.append((out, kd, vd))
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(30):
                out, (kd, vd) = chain(*sets[i])
            got[i] = (out, kd, vd)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


FIRST_CALL_CAPTURED = """
import torch
from forgeserve_b200 import ops, _lib as L
F8 = torch.float8_e4m3fn
k = torch.zeros(4, 2, 16, 128, dtype=torch.uint8, device="cuda").view(F8); v = torch.zeros_like(k.view(torch.uint8)).view(F8)
ks = torch.zeros(4, 2, 16, device="cuda"); vs = torch.zeros(4, 2, 16, device="cuda")
table = torch.tensor([[2]], device="cuda"); pos = torch.tensor([3], device="cuda")
qkv = torch.ones(1, 8 * 128, device="cuda", dtype=torch.bfloat16)
q = torch.empty(1, 512, device="cuda", dtype=torch.bfloat16); out = torch.empty_like(q)
d = ops.quant_paged_desc(k, v, ks, vs, table)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.rotary_kv_write(qkv, None, None, pos, d, 1, 1, 4, 2, 128, q_out=q)
    ops.attention_decode_quant(q, d, 16, pos, out, 1, 4, 2, 128)
g.replay(); torch.cuda.synchronize()
assert (q == 1).all() and torch.isfinite(out.float()).all() and k.view(torch.uint8)[2, :, 3].any(), out
assert L.device_error() == 0
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured():
    env = dict(os.environ, PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=240, env=env,
                       cwd=ROOT)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------------------- through the models

def model_pair(dtype, **kw):
    base = dict(vocab_size=64, d_model=64, n_layers=2, n_heads=4, n_kv_heads=2, max_seq_len=128)
    base.update(kw)
    cfg = ModelConfig(**base)
    torch.manual_seed(3)
    return cfg, ForgeModel(cfg).to(DEV, dtype).eval()


def logits64(m, cfg, idx, fake_quant=False):
    """The model's formulas in 64 bits (CPU): any rotary form, keys and values through e4m3 if asked."""
    w = {k: p.detach().double().cpu() for k, p in m.named_parameters()}
    B, T = idx.shape
    hd, nh, nkv = cfg.head_dim, cfg.n_heads, cfg.n_kv_heads
    cos, sin = (t.double()[:T] for t in (m._rope.cos, m._rope.sin))

    def norm(x, g):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.norm_eps) * g

    def turn(x):
        y, _ = rotate64(x.permute(1, 0, 2, 3).reshape(T, -1, hd), cos, sin, cfg.rope_layout)
        return y.view(T, B, -1, hd).permute(1, 0, 2, 3)

    def store(x):
        if not fake_quant:
            return x
        s = (x.abs().amax(-1, keepdim=True) / 448).clamp_min(2.0 ** -126)
        return (x / s).float().to(F8).double() * s

    x = w["tok_emb.weight"][idx]
    for i in range(cfg.n_layers):
        p = f"layers.{i}."
        h = norm(x, w[p + "attn_norm.weight"])
        q, k, v = (turn((h @ w[p + f"attn.w{n}.weight"].t()).view(B, T, -1, hd)) if n != "v" else
                   (h @ w[p + "attn.wv.weight"].t()).view(B, T, -1, hd) for n in "qkv")
        k, v = store(k), store(v)
        k, v = (t.repeat_interleave(nh // nkv, 2) for t in (k, v))
        s = torch.einsum("bthd,bshd->bhts", q, k) / math.sqrt(hd)
        s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -math.inf)
        x = x + torch.einsum("bhts,bshd->bthd", s.softmax(-1), v).reshape(B, T, -1) @ w[p + "attn.wo.weight"].t()
        h = norm(x, w[p + "mlp_norm.weight"])
        gate, up = h @ w[p + "mlp.w_gate.weight"].t(), h @ w[p + "mlp.w_up.weight"].t()
        x = x + (torch.nn.functional.silu(gate) * up) @ w[p + "mlp.w_down.weight"].t()
    return norm(x, w["norm.weight"]) @ w["tok_emb.weight"].t()


@pytest.mark.parametrize("kw", [dict(rope_layout="interleaved"), dict(rotary_dim=8), dict(rotary_dim=4, rope_layout="interleaved"),
                                dict(rope_scaling={"kind": "ntk", "factor": 4.0}),
                                dict(rope_scaling={"kind": "by_parts", "factor": 8.0, "original_max_len": 32,
                                                   "attn_factor": 1.2}, rope_layout="interleaved"),
                                dict(rope_scaling={"kind": "linear", "factor": 2.0}, rotary_dim=10)])
def test_model_with_rotary_forms(kw):
    """fp32 forward over a contiguous and a paged cache, in one piece and token by token, against 64 bits (the fp32
    parity bar, 1e-4)."""
    cfg, m = model_pair(torch.float32, **kw)
    idx = torch.randint(0, 64, (2, 24), generator=torch.Generator().manual_seed(1))
    want = logits64(m, cfg, idx)
    torch.testing.assert_close(m(idx).double().cpu(), want, atol=1e-4, rtol=1e-4)
    pool = PagedKVPool(cfg, 16, 4, device=DEV)
    table = torch.randperm(16, generator=torch.Generator().manual_seed(2))[:12].view(2, 6)
    pos = torch.arange(24).expand(2, 24)
    got = [m(idx[:, :20], pos[:, :20], pool.views(table, pos[:, :20]))]
    got += [m(idx[:, i: i + 1], pos[:, i: i + 1], pool.views(table, pos[:, i: i + 1])) for i in range(20, 24)]
    torch.testing.assert_close(torch.cat(got, 1).double().cpu(), want, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize("dtype,kw", [(torch.float32, {}), (torch.float32, dict(rope_layout="interleaved", rotary_dim=6)),
                                      (torch.bfloat16, dict(d_model=512, n_heads=4, n_kv_heads=2)),
                                      (torch.bfloat16, dict(d_model=256, n_heads=4, n_kv_heads=4, rope_layout="interleaved"))])
def test_model_over_an_8bit_pool(dtype, kw):
    """Prefill, a continued chunk and single tokens over an 8-bit pool. Codes may fall one step apart where a value lies
    next to a border, so the bar is on the distance to the 64-bit model with a quantised cache: it stays below the
    distance that the quantisation itself makes."""
    cfg, m = model_pair(dtype, **kw)
    idx = torch.randint(0, 64, (2, 30), generator=torch.Generator().manual_seed(1))
    plain, want = logits64(m, cfg, idx), logits64(m, cfg, idx, fake_quant=True)
    pool = PagedKVPool(cfg, 20, 4, dtype=F8, device=DEV)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:16].view(2, 8)
    pos = torch.arange(30).expand(2, 30)
    got = [m(idx[:, a:b], pos[:, a:b], pool.views(table, pos[:, a:b])) for a, b in [(0, 17), (17, 26)] + [(i, i + 1) for i in range(26, 30)]]
    got = torch.cat(got, 1).double().cpu()
    off, cost = (got - want).norm() / want.norm(), (plain - want).norm() / want.norm()
    assert cost > 0
    assert off <= (cost if dtype == torch.float32 else cost + 2.0 ** -6), (float(off), float(cost))


def test_view_update_over_an_8bit_pool():
    cfg, _ = model_pair(torch.float32)
    pool = PagedKVPool(cfg, 8, 4, dtype=F8, device=DEV)
    g = gen(3)
    k, v = (torch.randn(2, cfg.n_kv_heads, 9, cfg.head_dim, generator=g, device=DEV) for _ in range(2))
    pos = torch.arange(9).expand(2, 9)
    kd, vd = pool.views(torch.tensor([[1, 5, 2], [7, 0, 3]]), pos)[1].update(k, v)
    assert kd.shape == (2, cfg.n_kv_heads, 12, cfg.head_dim)
    for got, want in ((kd, k), (vd, v)):
        top = want.abs().amax(-1, keepdim=True)
        tol = torch.maximum(want.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10) * (1 + 2.0 ** -18)
        assert ((got[:, :, :9] - want).abs() <= tol).all() and not got[:, :, 9:].any()
    assert not pool.k[0].view(torch.uint8).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_engine_over_an_8bit_pool(dtype):
    """Graph replays, decode windows, eager steps and preemption give the same tokens over an 8-bit pool; greedy decode
    follows the pool's own prefill."""
    cfg, m = model_pair(dtype, d_model=256, n_heads=4, n_kv_heads=2)
    prompts = [[(7 * i + j) % 64 for j in range(3 + 5 * i)] for i in range(4)]

    def run(blocks=64, **kw):
        e = Engine(m, num_blocks=blocks, block_size=4, max_batch=4, kv_dtype=F8, **kw)
        assert e.pool.quantized
        for p in prompts:
            e.add_request(p, 20)
        return e.run(), e

    want, e = run(cuda_graphs=False)
    got, g = run()
    assert got == want and g.windows > 0
    # one request alone, in one row
    e1 = Engine(m, num_blocks=64, block_size=4, max_batch=1, kv_dtype=F8)
    rid = e1.add_request(prompts[2], 20)
    assert e1.run()[rid] == want[2]
    with pytest.raises(ValueError, match="kv_dtype"):
        Engine(m, 8, kv_dtype=torch.float16)


# --------------------------------------------------------------------- the same bits behind tables of any width

@pytest.mark.parametrize("dtype,nh,nkv,hd,bs", [(torch.bfloat16, 32, 8, 128, 16), (torch.float32, 8, 2, 64, 16),
                                                (torch.bfloat16, 40, 2, 256, 16), (torch.float32, 12, 12, 64, 20),
                                                (torch.float32, 20, 2, 128, 32), (torch.bfloat16, 8, 2, 80, 8),
                                                (torch.float32, 8, 2, 40, 16)])
def test_decode_bits_of_short_rows_do_not_depend_on_the_table(dtype, nh, nkv, hd, bs):
    """Rows of 1 to 512 visible slots behind a table of at most 512 (no join) and behind wider ones."""
    lengths = [1, 2, 17, 33, 100, 257, 500, 511, 512, 0]
    q, pools, table, positions, n_slots = decode_case(dtype, lengths, nh, nkv, hd, bs, seed=21)
    narrow = check_decode(q, pools, table, positions, 512, nh, nkv, hd)
    for times in (2, 9):
        wide = torch.cat([table] + [torch.zeros_like(table)] * (times - 1), 1)
        out = torch.full_like(q, 5.0)
        ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, wide), times * n_slots, positions, out, len(lengths),
                                   nh, nkv, hd)
        assert torch.equal(out, narrow), times
    # beside a long row
    long = torch.randint(0, pools[0].shape[0], (1, 3 * table.shape[1]), generator=gen(3), device=DEV)
    tables = torch.cat([torch.cat([table, table, table], 1), long])
    out = torch.empty(len(lengths) + 1, nh * hd, dtype=dtype, device=DEV)
    ops.attention_decode_quant(torch.cat([q, q[:1]]), ops.quant_paged_desc(*pools, tables), 3 * n_slots,
                               torch.cat([positions, positions.new_tensor([3 * n_slots - 1])]), out, len(lengths) + 1, nh,
                               nkv, hd)
    assert torch.equal(out[:-1], narrow)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_step_logits_do_not_depend_on_the_table(dtype):
    """A model's decode step over an 8-bit pool: an eager step's table and a captured graph's, padded to max_seq_len."""
    cfg, m = model_pair(dtype, d_model=256, n_heads=4, n_kv_heads=2, max_seq_len=2048)
    pool = PagedKVPool(cfg, 40, 16, dtype=F8, device=DEV)
    idx = torch.randint(0, 64, (3, 90), generator=torch.Generator().manual_seed(1))
    pos = torch.arange(90).expand(3, 90)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(2))[:18].view(3, 6)
    m(idx[:, :89], pos[:, :89], pool.views(table, pos[:, :89]))
    want = m(idx[:, 89:], pos[:, 89:], pool.views(table, pos[:, 89:]))
    wide = torch.cat([table, torch.zeros(3, 122, dtype=torch.int64)], 1)
    assert torch.equal(m(idx[:, 89:], pos[:, 89:], pool.views(wide, pos[:, 89:])), want)


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 8.0},
                                     {"kind": "by_parts", "factor": 8.0, "original_max_len": 64, "attn_factor": 1.2}])
def test_scaled_rotation_of_a_bf16_layer_rounds_once(scaling):
    """Whole heads in half layout with stretched positions over a plain cache: q and the stored k against 64 bits with one
    rounding, and q as over an 8-bit pool."""
    cfg, m = model_pair(torch.bfloat16, d_model=512, max_seq_len=1024, rope_scaling=scaling)
    a, hd, nh, nkv, bs = m.layers[0].attn, cfg.head_dim, cfg.n_heads, cfg.n_kv_heads, 16
    cos, sin = m._rope.on(torch.device(DEV))
    B, T = 2, 40
    pos = (torch.tensor([[3], [900]]) + torch.arange(T)).to(DEV)
    qkv = torch.randn(B * T, (nh + 2 * nkv) * hd, generator=gen(1), device=DEV).bfloat16()
    table = torch.arange(128, device=DEV).view(2, 64)
    qs = []
    for dtype in (torch.bfloat16, F8):
        pool = PagedKVPool(cfg, 128, bs, dtype=dtype, device=DEV)
        rows = qkv.clone()
        _rope_write(a, rows, cos, sin, pos, pool.views(table, pos)[0].descriptor(), B, T, 0, True)
        qs.append(rows[:, : nh * hd])
        if dtype == torch.bfloat16:
            k = pool.k[0]
    assert torch.equal(qs[0], qs[1])
    p = pos.view(-1)
    y, mag = rotate64(qkv.view(B * T, -1, hd).double()[:, : nh + nkv], cos.double()[p], sin.double()[p], "half")
    tol = HALF[torch.bfloat16] * y.abs() + 6 * U * mag
    assert ((qs[0].view(B * T, nh, hd).double() - y[:, :nh]).abs() <= tol[:, :nh]).all()
    row = torch.arange(B, device=DEV).repeat_interleave(T)
    got = k[table[row, p // bs], :, p % bs].double()
    assert ((got - y[:, nh:]).abs() <= tol[:, nh:]).all()


# ----------------------------------------------------------------------- small probabilities beside large ones

def far_ref(q, k, v, ks, vs, table, n, nh, nkv, hd):
    """(out, bound) of one row in 64 bits, as decode_ref, but with probabilities held to a fixed part of themselves down to
    2^-30 (bf16) or 2^-36 (fp32) of the largest p vs. A weight in f16, and fp32's remainder of it, is off by 2^-25 where
    f16's steps are smallest; the largest weight lies at 2^6 or above (fp32: 2^12), so that is 2^-31 (2^-37) of it, and one
    bit for the sum that it is divided by."""
    bs, rep, bf16 = k.shape[2], nh // nkv, q.dtype == torch.bfloat16
    t = torch.arange(n, device=DEV)
    blk, s = table[0][t // bs], t % bs
    kk, vv = (c.view(torch.uint8)[blk, :, s].view(F8).double().transpose(0, 1) for c in (k, v))
    ksr, vsr = ks[blk, :, s].double().t(), vs[blk, :, s].double().t()
    qq = q[0].double().view(nkv, rep, hd)
    p = torch.softmax(torch.einsum("grd,gnd->grn", qq, kk) * ksr[:, None] / math.sqrt(hd), -1)
    vd = vv * vsr[..., None]
    mag = torch.einsum("grd,gnd->grn", qq.abs(), kk.abs()) * ksr[:, None] / math.sqrt(hd)
    ds = (hd + 8) * U * mag.amax(-1)
    qerr = qq.abs().amax(-1) * 2.0 ** -25 * (kk.abs().sum(-1) * ksr).amax(-1)[:, None] / math.sqrt(hd) if bf16 else 0
    rel = 2 * (ds + qerr) + (2.0 ** -11 + 2.0 ** -12 if bf16 else 2.0 ** -21) + (n + 64) * U
    floor = (p * vsr[:, None]).amax(-1) * 2.0 ** (-30 if bf16 else -36) * vv.abs().sum(1).amax(-1)[:, None]
    out = torch.einsum("grn,gnd->grd", p, vd)
    bound = torch.einsum("grn,gnd->grd", p, vd.abs()) * rel[..., None] + floor[..., None]
    return out.reshape(1, -1), bound.reshape(1, -1)


def far_check(dtype, q, pools, table, n, nh, nkv, hd):
    out = torch.empty_like(q)
    ops.attention_decode_quant(q, ops.quant_paged_desc(*pools, table), n, torch.tensor([n - 1], device=DEV), out, 1, nh, nkv,
                               hd)
    want, bound = far_ref(q, *pools, table, n, nh, nkv, hd)
    tol = HALF[dtype] * (want.abs() + bound) + bound
    worst = ((out.double() - want).abs() / tol).max().item()
    assert worst <= 1, worst


FAR = [(torch.bfloat16, 8, 2, 128, 16), (torch.bfloat16, 8, 2, 64, 20), (torch.float32, 8, 2, 64, 16),
       (torch.float32, 4, 4, 128, 20), (torch.float32, 20, 2, 64, 16), (torch.bfloat16, 24, 2, 256, 16),
       (torch.float32, 4, 2, 256, 16), (torch.float32, 8, 2, 40, 16)]


@pytest.mark.parametrize("gap", [0, 14, 20, 25, 30])
@pytest.mark.parametrize("dtype,nh,nkv,hd,bs", FAR)
def test_decode_of_one_key_far_above_the_others(dtype, nh, nkv, hd, bs, gap):
    """A key 2^gap above 499 others, whose value is zero in half of the dims: there the others make the whole output."""
    n = 500
    q, pools, table, _, _ = decode_case(dtype, [n], nh, nkv, hd, bs, seed=31)
    k, v, ks, vs = pools
    ks.fill_(1.0)
    vs.fill_(1.0)
    codes = torch.zeros(k.shape, device=DEV)
    b, s = table[0, 70 // bs], 70 % bs
    codes[b, :, s, 0] = 1.0
    k.copy_(codes.to(F8))
    v.view(torch.uint8)[b, :, s, hd // 2:] = 0
    q.zero_().view(1, nh, hd)[:, :, 0] = gap * math.sqrt(hd) * math.log(2)
    far_check(dtype, q, pools, table, n, nh, nkv, hd)


@pytest.mark.parametrize("apart", [12, 20, 26])
@pytest.mark.parametrize("dtype,nh,nkv,hd,bs", FAR)
def test_decode_of_values_whose_scales_lie_far_apart(dtype, nh, nkv, hd, bs, apart):
    """Every other key's value 2^apart below its neighbours', in dims where those have zeros."""
    n = 500
    q, pools, table, _, _ = decode_case(dtype, [n], nh, nkv, hd, bs, seed=32)
    k, v, ks, vs = pools
    vs.fill_(1.0)
    t = torch.arange(n, device=DEV)
    b, s = table[0][t // bs], t % bs
    low = t % 2 == 1
    vs[b[low], :, s[low]] = 2.0 ** -apart
    raw = v.view(torch.uint8)
    raw[b[low], :, s[low], : hd // 2] = 0
    raw[b[~low], :, s[~low], hd // 2:] = 0
    far_check(dtype, q, pools, table, n, nh, nkv, hd)


def test_decode_of_one_key_far_above_a_long_row():
    """32 KV heads, 50000 keys 2^25 below one of them: a warp holds 768 keys of a split."""
    n, nh, nkv, hd, bs = 50000, 32, 32, 64, 64
    q, pools, table, _, _ = decode_case(torch.float32, [n], nh, nkv, hd, bs, seed=33)
    k, v, ks, vs = pools
    ks.fill_(1.0)
    vs.fill_(1.0)
    codes = torch.zeros(k.shape, device=DEV)
    b, s = table[0, 33000 // bs], 33000 % bs
    codes[b, :, s, 0] = 1.0
    k.copy_(codes.to(F8))
    v.view(torch.uint8)[:] &= 0x7F                                  # of one sign: lost ones are missed
    v.view(torch.uint8)[b, :, s, hd // 2:] = 0
    q.zero_().view(1, nh, hd)[:, :, 0] = 25 * math.sqrt(hd) * math.log(2)
    far_check(torch.float32, q, pools, table, n, nh, nkv, hd)


@pytest.mark.parametrize("hd", [128, 64, 80, 18])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_store_codes_beside_borders(dtype, hd):
    """The documented bounds: scales off by 2^-23 of top / 448, and codes those of x / scale or, where that lies within
    2^-21 of itself of a border between two codes, one of the two; over random rows and rows of values at and beside the
    borders. (1 / scale is off by 2 steps of 2^-23, its product with x by 2^-24: less than 2^-21.)"""
    T, nkv, bs = 400, 2, 16
    rows = torch.randn(T, 2 * nkv, hd, generator=gen(1), device=DEV) * torch.exp(
        3 * torch.randn(T, 2 * nkv, 1, generator=gen(2), device=DEV))
    steps = torch.arange(256, dtype=torch.uint8)
    values = steps.view(F8).float()
    values = values[torch.isfinite(values) & (steps < 128)]
    borders = ((values[1:] + values[:-1]) / 2).to(DEV)
    for r in range(0, T, 2):
        scale = 2.0 ** (r % 37 - 18) * (1 + (r * 0.37) % 1)
        pick = borders[torch.randint(0, borders.numel(), (2 * nkv, hd), generator=gen(r), device=DEV)] * scale
        up = torch.randint(-2, 3, pick.shape, generator=gen(r + 1), device=DEV)
        rows[r] = (pick.view(torch.int32) + up.int()).view(torch.float32)
        rows[r, :, 0] = 448 * scale
    x = rows.to(dtype)
    pools = quant_pool(T // bs + 1, nkv, bs, hd, 1)
    table = torch.randperm(T // bs + 1, generator=gen(4), device=DEV)[: T // bs][None]
    ops.rotary_kv_write(x.view(T, -1), None, None, torch.arange(T, device=DEV), ops.quant_paged_desc(*pools, table), 1, T, 0,
                        nkv, hd)
    t = torch.arange(T, device=DEV)
    for i, part in enumerate((x[:, :nkv], x[:, nkv:])):
        part = part.double().cpu()
        top = part.abs().amax(-1) / 448
        scale = pools[2 + i][table[0, t // bs], :, t % bs].cpu().double()
        assert ((scale - top).abs() <= 2.0 ** -23 * top).all()
        z = (part / scale[..., None]).abs().numpy()
        near, far = (torch.from_numpy((z * (1 + e)).astype(np.float32)).to(F8).float() for e in (-(2.0 ** -21), 2.0 ** -21))
        raw = bits(pools[i]).view(pools[i].shape)[table[0, t // bs], :, t % bs].cpu()
        got = raw.view(F8).float()
        assert ((near <= got.abs()) & (got.abs() <= far)).all()
        assert torch.equal(raw >= 128, torch.signbit(part))
        assert (near != far).any() or hd == 18


def test_pool_of_one_block_cut_from_a_larger_one():
    """k and its scales cut from a larger pool, v and its own: strides that differ in dimensions of one entry alone."""
    for nkv, bs in ((3, 32), (1, 1)):
        k, v, ks, vs = quant_pool(5, nkv + 1, bs, 64, 41)
        cut = [p[2:3, :nkv] for p in (k, v, ks, vs)]
        mixed = [cut[0], cut[1].contiguous(), cut[2], cut[3].contiguous()] if nkv == 1 else cut
        q = torch.randn(2, 2 * nkv * 64, generator=gen(42), device=DEV).bfloat16()
        table, n = torch.zeros(2, 1, dtype=torch.int64, device=DEV), bs
        pos = torch.tensor([n - 1, 0], device=DEV)
        got = check_decode(q, mixed, table, pos, n, 2 * nkv, nkv, 64)
        assert torch.equal(got, check_decode(q, [c.contiguous() for c in cut], table, pos, n, 2 * nkv, nkv, 64))
        kd, vd = ops.kv_dequant(ops.quant_paged_desc(*mixed, table), 2, n, nkv, 64, torch.float32)
        for d, c, s in ((kd, cut[0], cut[2]), (vd, cut[1], cut[3])):
            assert torch.equal(d[0], (c.float() * s[..., None])[0])


def test_model_over_an_8bit_pool_stays_near_the_quantised_model():
    """fp32: a code moves one step where rounding errors of some 2^-20 cross a border, one value in some 10^4, which makes
    about a hundredth of the quantisation's own distance; a quarter of that distance is allowed. bf16: whatever its own
    roundings do, the logits lie nearer to the model with a quantised cache than to the one without."""
    for dtype, kw in ((torch.float32, {}), (torch.float32, dict(rope_layout="interleaved", rotary_dim=6)),
                      (torch.float32, dict(rope_scaling={"kind": "ntk", "factor": 4.0})),
                      (torch.bfloat16, dict(d_model=512)), (torch.bfloat16, dict(d_model=256, n_kv_heads=4))):
        cfg, m = model_pair(dtype, **kw)
        idx = torch.randint(0, 64, (2, 30), generator=torch.Generator().manual_seed(1))
        plain, want = logits64(m, cfg, idx), logits64(m, cfg, idx, fake_quant=True)
        pool = PagedKVPool(cfg, 20, 4, dtype=F8, device=DEV)
        table = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:16].view(2, 8)
        pos = torch.arange(30).expand(2, 30)
        got = [m(idx[:, a:b], pos[:, a:b], pool.views(table, pos[:, a:b]))
               for a, b in [(0, 17), (17, 26)] + [(i, i + 1) for i in range(26, 30)]]
        got = torch.cat(got, 1).double().cpu()
        if dtype == torch.float32:
            assert (got - want).norm() <= 0.25 * (plain - want).norm(), kw
        else:
            assert (got - want).norm() < (got - plain).norm(), kw


REQUESTS = [([(7 * i + j) % 64 for j in range(3 + 5 * i)], 20) for i in range(4)]


def test_engine_preempts_over_an_8bit_pool():
    """A pool too small for its requests (fp32): blocks are taken back and used again with old codes and scales in them, and
    the tokens are those of a large pool. Each token is the best of a prefill of what came before over a fresh 8-bit
    pool, or within 2^-6 of the logits' spread of it (codes beside a border may differ)."""
    cfg, m = model_pair(torch.float32, d_model=256, n_heads=4, n_kv_heads=2)

    def run(blocks, **kw):
        e = Engine(m, num_blocks=blocks, block_size=4, max_batch=4, kv_dtype=F8, **kw)
        ids = [e.add_request(p, n) for p, n in REQUESTS]
        out = e.run()
        assert e.pool.allocator.num_free == blocks
        return [out[i] for i in ids], e.preemptions

    want, none = run(64, cuda_graphs=False)
    assert none == 0
    for kw in (dict(cuda_graphs=False), dict()):
        got, some = run(14, **kw)
        assert some > 0 and got == want, kw
    for (prompt, n), out in zip(REQUESTS, want):
        assert len(out) == n
        seq = prompt + out
        pool = PagedKVPool(cfg, 16, 4, dtype=F8, device=DEV)
        pos = torch.arange(len(seq))[None]
        logits = m(torch.tensor([seq]), pos, pool.views(torch.arange(-(-len(seq) // 4))[None], pos))[0]
        logits = logits[len(prompt) - 1: -1].double()
        spread = logits.amax(-1) - logits.amin(-1)
        chosen = logits.gather(1, torch.tensor(out, device=DEV)[:, None])[:, 0]
        assert (chosen >= logits.amax(-1) - 2.0 ** -6 * spread).all()


def pipeline_8bit_worker(rank, size, cfg_dict, sd, blocks, microbatches, pieces):
    from forgeserve_b200 import PipelineEngine, PipelineStage
    stage = PipelineStage(ModelConfig(**cfg_dict), rank, size)
    stage.load_from_full(sd)
    eng = PipelineEngine(stage.eval(), num_blocks=blocks, block_size=4, max_batch=4, microbatches=microbatches,
                         prefill_chunks=pieces, kv_dtype=F8)
    assert eng.pool.quantized and len(eng.pool.k) == len(stage.layers)
    ids = [eng.add_request(p, n) for p, n in REQUESTS]
    out = eng.run()
    return [out[i] for i in ids], eng.preemptions, eng.pool.allocator.num_free


@pytest.mark.parametrize("size,microbatches,pieces,blocks", [(2, 1, 1, 64), (2, 2, 1, 14), (3, 2, 3, 64)])
def test_pipeline_engine_over_8bit_pools(size, microbatches, pieces, blocks):
    """fp32 stages over 8-bit pools of their own layers give the Engine's tokens: prompts whole and in pieces, with
    preemption, in micro-batches."""
    from forgeserve_b200.tensor_parallel import run_in_threads
    cfg, m = model_pair(torch.float32, d_model=256, n_layers=3, n_heads=4, n_kv_heads=2)
    e = Engine(m, num_blocks=64, block_size=4, max_batch=4, kv_dtype=F8)
    ids = [e.add_request(p, n) for p, n in REQUESTS]
    out = e.run()
    sd = {k: t.detach().cpu() for k, t in m.state_dict().items()}
    for got, preemptions, free in run_in_threads(pipeline_8bit_worker, size, cfg.to_dict(), sd, blocks, microbatches, pieces):
        assert got == [out[i] for i in ids] and free == blocks
        assert (preemptions > 0) == (blocks == 14)


def stage_graph_worker(rank, size, cfg_dict, sd):
    from forgeserve_b200 import PipelineStage
    from forgeserve_b200.pipeline_engine import _StageDecodeGraph
    cfg = ModelConfig(**cfg_dict)
    stage = PipelineStage(cfg, rank, size)
    stage.load_from_full(sd)
    stage = stage.to(torch.bfloat16).eval()
    table = torch.randperm(16, generator=torch.Generator().manual_seed(2))[:12].view(3, 4)
    pos = torch.arange(60).expand(3, 60)
    idx = torch.randint(0, 64, (3, 60), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = []
    for graph in (False, True):
        pool = PagedKVPool(cfg, 16, 16, dtype=F8, device=DEV)
        views = pool.views(table, pos[:, :50])
        stage.run_layers_(stage.embed(idx[:, :50]), views[0].positions, views)
        g = _StageDecodeGraph(stage, pool, 3) if graph else None
        tokens = []
        for t in range(50, 60):
            if graph:
                tokens.append(g.run(pos[:, t: t + 1].to(DEV), table.to(DEV), idx[:, t]).clone())
            else:
                views = pool.views(table, pos[:, t: t + 1])
                x = stage.embed(idx[:, t: t + 1])
                stage.run_layers_(x, views[0].positions, views)
                tokens.append(ops.argmax(stage.head(x[:, -1:])[:, -1]))
        got.append((torch.stack(tokens), *[bits(t) for t in pool.k + pool.v + pool.k_scale + pool.v_scale]))
    torch.cuda.synchronize()
    return all(torch.equal(a, b) for a, b in zip(*got))


@torch.no_grad()
def test_stage_decode_graph_over_an_8bit_pool():
    """A stage's captured decode step, as decode windows replay it (its table padded to max_seq_len), gives the eager
    step's tokens and cache bit for bit."""
    from forgeserve_b200.tensor_parallel import run_in_threads
    cfg, m = model_pair(torch.float32, d_model=256, n_heads=4, n_kv_heads=2, max_seq_len=1024)
    sd = {k: t.detach().cpu() for k, t in m.state_dict().items()}
    assert run_in_threads(stage_graph_worker, 1, cfg.to_dict(), sd) == [True]


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 16), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("kind", ["plain", "8-bit"])
def test_tables_padded_with_no_block(kind, dtype, hd):
    """Columns past a row's last token may hold anything, -1 or a number past the pool, in a prompt, a continued chunk
    and a decode step: the same logits as with block 0 there, and nothing is flagged (the fixture looks)."""
    cfg, m = model_pair(dtype, d_model=4 * hd, max_seq_len=512)
    idx = torch.randint(0, 64, (2, 100), generator=torch.Generator().manual_seed(1))
    pos = torch.arange(100).expand(2, 100)
    blocks = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:14].view(2, 7)
    got = []
    for pad in (0, -1, 1 << 40):
        pool = PagedKVPool(cfg, 20, 16, dtype=F8 if kind == "8-bit" else dtype, device=DEV)
        table = torch.cat([blocks, torch.full((2, 20), pad)], 1)
        logits = []
        for a, b in ((0, 70), (70, 99), (99, 100)):
            t = table.clone()
            t[:, -(-b // 16):] = pad                                # blocks not granted yet
            logits.append(m(idx[:, a:b], pos[:, a:b], pool.views(t, pos[:, a:b])))
        got.append(torch.cat(logits, 1))
        assert L.device_error() == 0, pad
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtype", [F8, torch.float32])
def test_tables_of_more_rows_than_the_step(dtype):
    """A step takes the first rows of a table that has more; one of fewer rows is refused over an 8-bit pool."""
    cfg, m = model_pair(torch.float32)
    idx = torch.randint(0, 64, (2, 9), generator=torch.Generator().manual_seed(1))
    pos = torch.arange(9).expand(2, 9)
    table = torch.arange(15).view(5, 3)
    got = []
    for t in (table, table[:2]):
        pool = PagedKVPool(cfg, 16, 4, dtype=dtype, device=DEV)
        a = m(idx[:, :8], pos[:, :8], pool.views(t, pos[:, :8]))
        got.append(torch.cat([a, m(idx[:, 8:], pos[:, 8:], pool.views(t, pos[:, 8:]))], 1))
    assert torch.equal(*got)
    if dtype == F8:
        with pytest.raises(ValueError, match="rows"):
            m(idx, pos, pool.views(table[:1], pos))


@pytest.mark.parametrize("hd", [128, 18])
def test_dequant_for_queries_flags_what_they_see(hd):
    """Bad blocks: of a row that no query sees, of rows whose first, middle or last query reaches them, or ends one slot
    before."""
    bs, T = 4, 3
    k, v, ks, vs = quant_pool(6, 2, bs, hd, 9)
    table = torch.tensor([[1, -1, 99, 2], [3, 4, 5, -7]], device=DEV)
    desc = ops.quant_paged_desc(k, v, ks, vs, table)
    plain, _ = ops.kv_dequant(desc, 2, 16, 2, hd, torch.float32)
    assert L.device_error(clear=True) == L.FS_ERR_BAD_SLOT
    for pos, bad in (([[0, 1, 3], [9, 10, 11]], False), ([[0, 1, 4], [0, 0, 0]], True), ([[4, 1, 0], [0, 0, 0]], True),
                     ([[-1, -1, -1], [0, 12, 3]], True), ([[-1, 3, -1], [11, 0, 0]], False),
                     ([[0, 0, 0], [0, 0, 1000]], True)):
        kd, vd = ops.kv_dequant(desc, 2, 16, 2, hd, torch.float32, torch.tensor(pos, device=DEV))
        assert L.device_error(clear=True) == (L.FS_ERR_BAD_SLOT if bad else 0), pos
        assert torch.equal(kd, plain) and not vd[0, :, 4:12].any() and not vd[1, :, 12:].any()
    for pos in (torch.zeros(2, 0, dtype=torch.int64, device=DEV), torch.zeros(3, 2, dtype=torch.int64, device=DEV),
                torch.zeros(2, 3, device=DEV)):
        with pytest.raises(ValueError, match="positions"):
            ops.kv_dequant(desc, 2, 16, 2, hd, torch.float32, pos)


@torch.no_grad()
def test_captured_chunk_over_an_8bit_pool():
    """A step of several tokens captured once over views of static tables and positions, replayed as both move on."""
    cfg, m = model_pair(torch.float32)
    idx = torch.randint(0, 64, (1, 40), generator=torch.Generator().manual_seed(1)).to(DEV)
    pos = torch.arange(40, device=DEV)[None]
    blocks = torch.randperm(12, generator=torch.Generator().manual_seed(2))[:10].to(DEV)
    want_pool, pool = (PagedKVPool(cfg, 12, 4, dtype=F8, device=DEV) for _ in range(2))
    cos, sin = m._rope.on(torch.device(DEV))

    def step(tokens, positions, views):
        x = ops.embed(tokens, m.tok_emb.weight)
        for blk, view in zip(m.layers, views):
            layer_forward_(blk, x, positions, view, cos, sin)
        return x

    cuts = [slice(a, a + 4) for a in range(0, 40, 4)]
    want = [step(idx[:, c], pos[:, c].contiguous(), want_pool.views(blocks[None], pos[:, c])) for c in cuts]
    toks, p, table = idx[:, :4].clone(), pos[:, :4].clone(), torch.full((1, 10), -1, device=DEV)
    table[0, 0] = blocks[0]
    views = pool.views(table, p)
    assert views[0].tables.data_ptr() == table.data_ptr() and views[0].positions.data_ptr() == p.data_ptr()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(toks, p, views)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = step(toks, p, views)
    for i, c in enumerate(cuts):
        toks.copy_(idx[:, c])
        p.copy_(pos[:, c])
        table[0, i] = blocks[i]
        g.replay()
        assert torch.equal(out, want[i]), i
    assert torch.equal(bits(pool.k[1][blocks]), bits(want_pool.k[1][blocks]))
