"""The 8-bit page cache on a B200 against its plain 64-bit restatement: slot maps, append, decode attention."""
import numpy as np
import pytest
import torch

import kv8_cases as plain
from conftest import pkg

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ slot map


def map_case(rng, B, width, ctx_max, new_max, supply_extra=0):
    ctx = [int(c) for c in rng.integers(0, ctx_max + 1, B)]
    new = [int(n) for n in rng.integers(0, new_max + 1, B)]
    have = [-(-c // 16) for c in ctx]
    need = sum(max(0, -(-(c + n) // 16) - h) for c, n, h in zip(ctx, new, have) if c + n <= width * 16)
    blocks = sum(have) + need + supply_extra + 3
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((B, width), -7, dtype=np.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    return ctx, new, table, [int(i) for i in ids], at, blocks


def check_map(ops, ctx, new, table, supply, used, rows, blocks, code=0):
    t, status, given = torch.from_numpy(table.copy()).to(DEV), status_word(), ints([used])
    m = ops.kv_slot_map(ints(ctx), ints(new), t, ints(supply), given, rows, blocks, status=status)
    want = table.copy()
    lens, start, seq, pos, slot, n_used = plain.slot_map(ctx, new, want, supply, used, rows, blocks)
    assert m.lens.tolist() == lens and m.row_start.tolist() == start and m.supply_used.tolist() == [n_used]
    assert m.row_seq.tolist() == seq and m.positions.tolist() == pos and m.slots.tolist() == slot
    assert np.array_equal(t.cpu().numpy(), want)
    assert status.item() == code and given.item() == used


@pytest.mark.parametrize("B,width,ctx_max,new_max", [(1, 1, 0, 16), (1, 40, 200, 400), (3, 4, 30, 2), (37, 30, 300, 1), (256, 40, 500, 1),
                                                     (257, 20, 100, 200), (700, 9, 60, 70), (4096, 3, 20, 20)])
def test_slot_map(ops, B, width, ctx_max, new_max):
    rng = np.random.default_rng(B)
    ctx, new, table, supply, used, blocks = map_case(rng, B, width, ctx_max, new_max)
    total = sum(new)
    for rows in (total, total + 1 + B):
        check_map(ops, ctx, new, table, supply, used, rows, blocks)


def test_slot_map_of_a_decode_step_at_every_offset(ops):
    ctx = list(range(0, 49))
    table = np.arange(49 * 4, dtype=np.int32).reshape(49, 4)
    check_map(ops, ctx, [1] * 49, table, list(range(1000, 1010)), 2, 64, 2000)


def test_slot_map_without_new_tokens_or_rows(ops):
    check_map(ops, [5, 0], [0, 0], np.array([[3], [4]], dtype=np.int32), [], 0, 0, 9)
    check_map(ops, [5, 0], [0, 0], np.array([[3], [4]], dtype=np.int32), [], 0, 3, 9)


def test_slot_map_findings(ops):
    BAD_ID, BAD_LEN, NO_PAGES = 16, 17, 21
    table = np.array([[3, -1, -1], [4, -1, -1]], dtype=np.int32)
    check_map(ops, [16, 1], [32, 40], table, [5, 6, 7], 0, 80, 9, code=NO_PAGES)     # pages for the first, one for the second
    check_map(ops, [16, 1], [1, 1], table, [5, 6, 7], 4, 4, 9, code=NO_PAGES)        # more used than there are
    check_map(ops, [16, 1], [1, 1], table, [5, 6, 7], -1, 4, 9, code=NO_PAGES)
    check_map(ops, [16, 1], [1, 1], table, [99, 6, 7], 0, 4, 9, code=BAD_ID)         # a free page that is no page
    check_map(ops, [15, 1], [1, 1], np.array([[-1, -1], [4, -1]], dtype=np.int32), [5], 0, 2, 9, code=BAD_ID)
    check_map(ops, [16, 1], [33, 2], table, [5, 6, 7], 0, 4, 9, code=BAD_LEN)        # wider than the table
    check_map(ops, [-1, 1], [3, 2], table, [5, 6, 7], 0, 4, 9, code=BAD_LEN)
    check_map(ops, [49, 1], [0, 2], table, [5, 6, 7], 0, 4, 9, code=BAD_LEN)
    check_map(ops, [16, 1], [2 ** 31 - 1, 2], table, [5, 6, 7], 0, 4, 9, code=BAD_LEN)
    check_map(ops, [16, 1], [4, 4], table, [5, 6, 7], 0, 5, 9, code=BAD_LEN)         # more tokens than rows


# -------------------------------------------------------------------- append


def check_append(ops, rows, slots, codes, exps, dtype, kv=None, code=0):
    """rows: (k, v) float32 arrays [R, H, D] already exact in dtype; the caches of both start from `codes` and `exps`."""
    k, v = (torch.from_numpy(r).to(DEV, dtype) for r in rows) if kv is None else kv
    pools = [plain.pool_of(codes.copy()), plain.pool_of(codes[::-1].copy())]
    scales = [plain.scale_of(exps), plain.scale_of(exps[::-1].copy())]
    for _ in range(2):  # the same call again changes nothing
        status = status_word()
        ops.kv8_append(k, v, *pools, *scales, ints(slots), status=status)
        assert status.item() == code
        good = [s if s < codes.shape[0] * 16 else -1 for s in slots]
        for x, pool, scale, c, e in zip((k, v), pools, scales, (codes, codes[::-1]), (exps, exps[::-1])):
            want, want_e = c.copy(), e.copy()
            plain.append(x.double().cpu().numpy(), good, want, want_e)
            got = pool.view(torch.uint8).cpu().numpy()
            assert np.array_equal(scale.view(torch.uint8).cpu().numpy().astype(int) - 127, want_e)
            # all bytes, those of slots that no row names included; NaN has two codes
            assert np.array_equal(np.where(got & 127 == 127, 127, got), np.where(want & 127 == 127, 127, want))


def rows_of(rng, R, H, D, dtype, grow=1.0):
    x = [(rng.standard_normal((R, H, D)) * np.exp(rng.uniform(-grow, grow, (R, H, 1)))).astype(np.float32) for _ in range(2)]
    return [torch.from_numpy(a).to(dtype).float().numpy() for a in x]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D", [(4, 128), (2, 64), (1, 128), (3, 64), (8, 128)])
def test_append_of_single_tokens(ops, dtype, H, D):
    rng = np.random.default_rng(H * D)
    codes, exps = plain.random_cache(rng, 40, H, D, spread=4)
    pages = rng.permutation(40)[:33]
    slots = [int(p) * 16 + i % 16 for i, p in enumerate(pages)]
    slots[5] = slots[11] = -1
    check_append(ops, rows_of(rng, 33, H, D, dtype, grow=4.0), slots, codes, exps, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D,lens", [(4, 128, [(0, 16), (3, 40), (15, 2), (0, 1), (7, 9)]), (2, 64, [(5, 100), (0, 333)]), (2, 128, [(9, 700), (1, 1400)]),
                                      (1, 64, [(13, 9000)])])
def test_append_of_prompts(ops, dtype, H, D, lens):
    rng = np.random.default_rng(len(lens))
    blocks = sum(-(-(c + n) // 16) for c, n in lens) + 2
    codes, exps = plain.random_cache(rng, blocks, H, D)
    ids, slots = [int(p) for p in rng.permutation(blocks)], []
    for c, n in lens:
        own = [ids.pop() for _ in range(-(-(c + n) // 16))]
        slots += [own[p // 16] * 16 + p % 16 for p in range(c, c + n)] + [-1] * (n % 3)
    check_append(ops, rows_of(rng, len(slots), H, D, dtype), slots, codes, exps, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_at_the_ends_of_the_range(ops, dtype):
    rng = np.random.default_rng(3)
    H, D = 2, 64
    codes, exps = plain.random_cache(rng, 24, H, D)
    codes[20, :, :3] = 127  # NaN among the earlier rows stays NaN when they are rounded again
    k, v = rows_of(rng, 12, H, D, dtype)
    for x in (k, v):
        x[0] = 0.0                         # nothing but zeros
        x[1, 0, 3], x[1, 1, 4] = np.inf, np.nan
        x[2] = np.nan                      # nothing finite
        x[3] *= 2.0 ** 40                  # above the largest scale: 448 * 2^31
        x[4] *= 2.0 ** -50                 # below the smallest
        x[5, 0] = 448.0
        x[5, 1] = 1.75 * 2.0 ** -20
        x[6, 0, :] = 0.0
        x[6, 0, 7] = torch.tensor(450.0).to(dtype).item()
        x[7] = 1e-40
        x[8] *= 2.0 ** 9                   # makes the scale of a page with tokens grow by a lot
        x[9] *= 2.0 ** 30
    exps[20] = -9
    exps[21] = 31
    exps[22] = 90                          # bytes beyond the range are taken for the nearest
    exps[23] = -100
    slots = [p * 16 for p in range(8)] + [20 * 16 + 5, 21 * 16 + 1, 22 * 16 + 2, 23 * 16 + 3]
    check_append(ops, (k, v), slots, codes, exps, dtype)


def test_append_of_a_slot_named_more_than_once(ops):
    """Padding rows of a pass all go to slot 0 of a scratch page; the last one stays."""
    rng = np.random.default_rng(4)
    codes, exps = plain.random_cache(rng, 6, 2, 128)
    slots = [3 * 16 + 2, 3 * 16 + 3, 3 * 16 + 3] + [5 * 16] * 45 + [2 * 16 + 9] * 17 + [16 + i for i in range(16)] * 2
    check_append(ops, rows_of(rng, len(slots), 2, 128, torch.bfloat16), slots, codes, exps, torch.bfloat16)


def test_append_of_strided_rows_and_slots_that_are_none(ops):
    rng = np.random.default_rng(5)
    H, D, R = 4, 128, 50
    codes, exps = plain.random_cache(rng, 20, H, D)
    fused = torch.from_numpy(rng.standard_normal((R, 16 + 2 * H, D)).astype(np.float32)).to(DEV, torch.bfloat16)
    slots = [int(p) * 16 + int(rng.integers(16)) for p in rng.permutation(20)] + [20 * 16, 2 ** 31 - 1, -1, -2 ** 31] + [-1] * 26
    check_append(ops, None, slots, codes, exps, torch.bfloat16, kv=(fused[:, 16:16 + H], fused[:, 16 + H:]), code=16)


def test_append_of_a_single_row_of_any_stride(ops):
    """One row may be a view whose row stride is no multiple of anything: it says nothing."""
    rng = np.random.default_rng(36)
    codes, exps = plain.random_cache(rng, 3, 2, 64)
    kv = [torch.from_numpy(rng.standard_normal((1, 2, 64)).astype(np.float32)).to(DEV).as_strided((1, 2, 64), (stride, 64, 1)) for stride in (3, 1001)]
    check_append(ops, None, [21], codes, exps, torch.float32, kv=kv)


def test_wrappers_refuse(ops):
    pools = ops.kv8_pools(4, 2, 64, DEV)
    x, slots = torch.zeros(3, 2, 64, device=DEV), ints([0, 1, 2])
    for bad in (dict(k_new=x.half()), dict(k_new=x.bfloat16()), dict(v_new=x[:2]), dict(slots=slots.long()), dict(slots=slots[:2]), dict(k_new=x[:1].expand(3, 2, 64)),
                dict(k_new=x.transpose(0, 1).reshape(3, 2, 64).transpose(1, 2).contiguous().transpose(1, 2)), dict(k_pool=pools[0].view(torch.uint8)),
                dict(v_pool=pools[1][:3]), dict(k_scale=pools[2].view(torch.uint8)), dict(v_scale=pools[3][:, :1]), dict(slots=slots.cpu()),
                dict(status=torch.zeros(1, dtype=torch.int32)), dict(status=torch.zeros(0, dtype=torch.int32, device=DEV))):
        args = dict(k_new=x, v_new=x, k_pool=pools[0], v_pool=pools[1], k_scale=pools[2], v_scale=pools[3], slots=slots) | bad
        with pytest.raises(ValueError):
            ops.kv8_append(**args)
    q, table = torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16), ints([[0], [1], [2]])
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32].contiguous()), dict(q=q.transpose(0, 1)), dict(block_table=table[:2]), dict(ctx_lens=slots[:2]),
                dict(out=q[:2]), dict(out=q.float()), dict(ctx_lens=slots.cpu()), dict(workspace=torch.zeros(1 << 16))):
        args = dict(q=q, k_pool=pools[0], v_pool=pools[1], k_scale=pools[2], v_scale=pools[3], block_table=table, ctx_lens=slots, scale=0.1) | bad
        with pytest.raises(ValueError):
            ops.kv8_attn_decode(**args)
    err = pkg("_lib").B200Error
    with pytest.raises(err, match="workspace"):
        ops.kv8_attn_decode(q, *pools, table, slots, 0.1, workspace=torch.zeros(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(err, match="scale"):
        ops.kv8_attn_decode(q, *pools, table, slots, -0.1)
    with pytest.raises(err, match="multiple of kv heads"):
        ops.kv8_attn_decode(q[:, :3].contiguous(), *pools, table, slots, 0.1)
    for call in (lambda: ops.kv8_append(None, x, *pools, slots), lambda: ops.kv8_append(x, x, *pools, [0, 1, 2]),
                 lambda: ops.kv_slot_map(slots, slots, table, slots, slots[:1], -1, 4), lambda: ops.kv_slot_map(slots, slots, table, slots, slots, 1, 4),
                 lambda: ops.kv_slot_map(slots, slots[:2], table, slots, slots[:1], 1, 4), lambda: ops.kv_slot_map(slots, slots, table, slots, slots[:1], 2 ** 40, 4)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.kv8_attn_decode(q, *pools, table, slots, "0.1")
    odd = torch.zeros(17, device=DEV, dtype=torch.uint8)[1:9].view(4, 2).view(ops.KV8_SCALE_DTYPE)
    with pytest.raises(err, match="aligned"):
        ops.kv8_attn_decode(q, pools[0], pools[1], odd, pools[3], table, slots, 0.1)
    with pytest.raises(err, match="dimension"):
        ops.kv_slot_map(slots, slots, table, slots, slots[:1], 4, 0)
    ops.kv8_append(x[:0], x[:0], *pools, slots[:0])
    assert ops.kv8_attn_decode(q[:0], *pools, table[:0], slots[:0], 0.1).shape == (0, 4, 64)


# -------------------------------------------------------------------- decode


def attn_case(rng, lens, Hq, H, D, spread=3, q_size=1.0, width=None):
    blocks = sum(-(-L // 16) for L in lens) + 3
    kc, ke = plain.random_cache(rng, blocks, H, D, spread)
    vc, ve = plain.random_cache(rng, blocks, H, D, spread)
    ids = [int(i) for i in rng.permutation(blocks)]
    table = np.full((len(lens), width or max(1, max(-(-L // 16) for L in lens)) + 1), -1, dtype=np.int32)
    for b, L in enumerate(lens):
        for p in range(-(-L // 16)):
            table[b, p] = ids.pop()
        if L % 16:  # behind the last token
            kc[table[b, L // 16], :, L % 16:] = 127
            vc[table[b, L // 16], :, L % 16:] = 255
    q = torch.from_numpy((rng.standard_normal((len(lens), Hq, D)) * q_size).astype(np.float32)).bfloat16()
    return q, kc, ke, vc, ve, table


def rows_at(codes, exps, row, L):
    p = row[:-(-L // 16)]
    x = plain.decode(codes[p]) * 2.0 ** np.clip(exps[p], -32, 31)[:, :, None, None]
    return x.transpose(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:L]


def check_attn(got, q, kc, ke, vc, ve, table, lens, scale, q_step=0.0):
    got = got.double().cpu().numpy()
    for b, L in enumerate(lens):
        unit = np.repeat(2.0 ** np.clip(ve[table[b][:-(-L // 16)]], -32, 31), 16, axis=0)[:L]
        want, tol = plain.attention(q[b].double().numpy(), rows_at(kc, ke, table[b], L), rows_at(vc, ve, table[b], L), unit, scale, q_step)
        over = np.abs(got[b] - want) - tol
        assert np.isfinite(got[b]).all() and over.max() <= 0, (b, L, float(over.max()), float(np.abs(want).max()))


def run_decode(ops, q, kc, ke, vc, ve, table, lens, scale, split=0):
    q = q.to(DEV)
    ws = ops.kv8_attn_workspace(len(lens), q.shape[1], kc.shape[1], q.shape[2], table.shape[1], DEV, split)
    out = ops.kv8_attn_decode(q, plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table).to(DEV),
                              ints(lens), scale, split_tokens=split, workspace=ws, out=torch.full_like(q, float("nan")))
    ops.read_status(ws, "kv8_attn_decode")
    return out


@pytest.mark.parametrize("Hq,H,D", [(32, 4, 128), (64, 4, 128), (8, 2, 64), (16, 2, 64), (4, 4, 128), (7, 1, 128), (12, 1, 64), (24, 3, 64), (8, 8, 128),
                                    (96, 8, 64), (128, 8, 128), (40, 1, 128), (100, 2, 64), (18, 2, 128), (1, 1, 64)])
def test_decode_heads(ops, Hq, H, D):
    rng = np.random.default_rng(Hq * H + D)
    lens = [1, 15, 0, 16, 17, 33, 200, 531]
    case = attn_case(rng, lens, Hq, H, D)
    for split in (0, 16, 64, 1024):
        check_attn(run_decode(ops, *case, lens, D ** -0.5, split), *case, lens, D ** -0.5)


@pytest.mark.parametrize("H,D", [(4, 128), (2, 64), (1, 128), (8, 64)])
@pytest.mark.parametrize("spread,q_size,scale", [(0, 1.0, 0.1), (20, 1.0, 0.1), (3, 30.0, 1.0), (3, 1e-30, 1.0), (3, 1e20, 1e-20), (25, 1e-6, 1.0)])
def test_decode_magnitudes(ops, H, D, spread, q_size, scale):
    """Pages whose scales differ by up to 2^50, sharp and flat weights, queries at the ends of bf16."""
    rng = np.random.default_rng(7 + spread)
    lens = [64, 100, 1, 700]
    case = attn_case(rng, lens, 4 * H, H, D, spread, q_size)
    check_attn(run_decode(ops, *case, lens, scale, 128), *case, lens, scale)


def test_decode_scale_bytes_beyond_the_range(ops):
    rng = np.random.default_rng(9)
    lens = [50, 90]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, 8, 2, 64)
    ke[table[0, 0]], ve[table[1, 2]], ve[table[1, 1]] = -127, 128, -90
    check_attn(run_decode(ops, q, kc, ke, vc, ve, table, lens, 1e-12), q, kc, ke, vc, ve, table, lens, 1e-12)


@pytest.mark.parametrize("B,top", [(1, 20011), (3, 6000), (70, 900), (300, 130), (5000, 40)])
def test_decode_batches(ops, B, top):
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, top + 1, B)]
    lens[0] = top
    case = attn_case(rng, lens, 8, 2, 128)
    check_attn(run_decode(ops, *case, lens, 0.09), *case, lens, 0.09)


def test_decode_one_workspace_for_many_shapes(ops):
    """Calls of other sizes and head shapes take turns with a workspace; parts of rows are counted in it."""
    rng = np.random.default_rng(14)
    shapes = [(8, 2, 64, [3000]), (32, 4, 128, [100, 700, 30]), (8, 2, 64, [900] * 40), (16, 1, 128, [2000, 0, 17, 5]), (32, 4, 128, [2500] * 9)]
    cases = [attn_case(rng, lens, Hq, H, D, width=200) for Hq, H, D, lens in shapes]
    n = max(ops.kv8_attn_workspace(len(lens), Hq, H, D, 200, DEV).numel() for Hq, H, D, lens in shapes)
    ws = torch.zeros(n, dtype=torch.uint8, device=DEV)
    first = []
    for turn in range(3):
        for i, (q, kc, ke, vc, ve, table) in enumerate(cases):
            lens = shapes[i][3]
            out = ops.kv8_attn_decode(q.to(DEV), plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table).to(DEV),
                                      ints(lens), 0.1, workspace=ws)
            if turn == 0:
                check_attn(out, q, kc, ke, vc, ve, table, lens, 0.1)
                first.append(out)
            assert torch.equal(out, first[i])
    ops.read_status(ws, "turns")


@pytest.mark.parametrize("lens", [[0, 0, 0], [0] * 300 + [33] + [0] * 300, [1] * 700, [16] * 37 + [0, 4000, 0] + [1] * 5, [5000] + [0] * 20, [15, 16, 17] * 333])
def test_decode_runs_over_rows_of_all_lengths(ops, lens):
    rng = np.random.default_rng(len(lens))
    case = attn_case(rng, lens, 8, 2, 64)
    for split in (0, 16):
        check_attn(run_decode(ops, *case, lens, 0.1, split), *case, lens, 0.1)


def test_decode_values_of_nan_and_what_they_reach(ops):
    rng = np.random.default_rng(11)
    lens = [40, 40]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, 8, 2, 64)
    vc[table[0, 1], 1, 3, 5] = 127   # a value of kv head 1, column 5
    kc[table[1, 0], 0, 2, 7] = 255   # a key of kv head 0
    out = run_decode(ops, q, kc, ke, vc, ve, table, lens, 0.1).isnan().cpu()
    want = torch.zeros(2, 8, 64, dtype=torch.bool)
    want[0, 4:, 5] = True
    want[1, :4] = True
    assert torch.equal(out, want)


def test_decode_findings(ops):
    rng = np.random.default_rng(12)
    lens = [40, 40]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, 8, 2, 64)
    for bad, code in ((10 ** 6, "pool"), (-1, "pool")):
        t = table.copy()
        t[1, 2] = bad
        with pytest.raises(pkg("_lib").B200Error, match=code):
            run_decode(ops, q, kc, ke, vc, ve, t, lens, 0.1)
    for bad in (-1, 16 * table.shape[1] + 1):
        t = np.where(table < 0, 0, table)
        with pytest.raises(pkg("_lib").B200Error, match="length"):
            run_decode(ops, q, kc, ke, vc, ve, t, [40, bad], 0.1)


def test_decode_pages_past_32_bits_of_bytes(ops):
    """A pool of 4.5 GB: its last pages are more than 2^32 bytes from its first."""
    D, H, blocks = 128, 4, 560_000
    pools = [torch.zeros(blocks, H, 16, D, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.full((blocks, H), 120, dtype=torch.uint8, device=DEV) for _ in range(2)]
    cache = [p.view(plain.E4M3) for p in pools] + [s.view(plain.E8M0) for s in scales]
    rng = np.random.default_rng(13)
    slots = [(blocks - 1) * 16 + i for i in range(16)] + [i for i in range(16)] + [(blocks - 5) * 16 + i for i in range(9)]
    k, v = (torch.from_numpy(r).to(DEV, torch.bfloat16) for r in rows_of(rng, len(slots), H, D, torch.bfloat16))
    ops.kv8_append(k, v, *cache, ints(slots))
    q = torch.randn(1, 32, D, device=DEV).bfloat16()
    table = ints([[blocks - 1, 0, blocks - 5]])
    got = ops.kv8_attn_decode(q, *cache, table, ints([41]), 0.1)
    small = [torch.cat([c.view(torch.uint8)[blocks - 1:], c.view(torch.uint8)[:1], c.view(torch.uint8)[blocks - 5:blocks - 4]]).view(c.dtype) for c in cache]
    assert torch.equal(got, ops.kv8_attn_decode(q, *small, ints([[0, 1, 2]]), ints([41]), 0.1))
    check_attn(got, q.cpu(), *(f(c) for c in (small[0], small[2], small[1], small[3]) for f in [lambda c: c.view(torch.uint8).cpu().numpy()
               if c.dtype == plain.E4M3 else c.view(torch.uint8).cpu().numpy().astype(int) - 127]), np.array([[0, 1, 2]]), [41], 0.1)
    q = torch.randn(5, 32, D, device=DEV).bfloat16()
    assert torch.equal(ops.kv8_attn_prefill(q, *cache, table[0], 36, 0.1), ops.kv8_attn_prefill(q, *small, ints([0, 1, 2]), 36, 0.1))


@pytest.mark.parametrize("Hq,H,D", [(32, 4, 128), (5, 1, 64)])
def test_pages_that_rows_share_or_name_twice(ops, Hq, H, D):
    """Rows with common pages ahead of their own, a row that is another one again, a row that names a page three times."""
    rng = np.random.default_rng(37)
    q, kc, ke, vc, ve, table = attn_case(rng, [160, 40, 40, 64], Hq, H, D)
    table[1, :2], table[2], table[3, :4] = table[0, :2], table[1], table[0, [5, 5, 2, 5]]
    lens = [160, 40, 40, 64]
    out = run_decode(ops, q, kc, ke, vc, ve, table, lens, 0.1)
    check_attn(out, q, kc, ke, vc, ve, table, lens, 0.1)
    q = torch.from_numpy(rng.standard_normal((20, Hq, D)).astype(np.float32)).bfloat16()
    got = ops.kv8_attn_prefill(q.to(DEV), plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), ints(table[3].tolist()), 44, 0.1)
    check_attn(got, q, kc, ke, vc, ve, [table[3]] * 20, range(45, 65), 0.1, 2.0 ** -10 / 224)


def test_attention_in_place(ops):
    """The output may be the queries' own memory: a query is read before anything is written over it."""
    rng = np.random.default_rng(38)
    lens = [700, 0, 33, 1, 2500]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, 12, 4, 128)
    cache = [plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve)]
    table, lens = torch.from_numpy(table).to(DEV), ints(lens)
    want, q = ops.kv8_attn_decode(q.to(DEV), *cache, table, lens, 0.1), q.to(DEV)
    assert ops.kv8_attn_decode(q, *cache, table, lens, 0.1, out=q) is q and torch.equal(q, want)
    for n, first in ((300, 400), (9, 2400)):
        row = table[0 if first == 400 else 4]
        q = torch.from_numpy(rng.standard_normal((n, 12, 128)).astype(np.float32)).to(DEV, torch.bfloat16)
        want = ops.kv8_attn_prefill(q, *cache, row, first, 0.1)
        assert torch.equal(ops.kv8_attn_prefill(q, *cache, row, first, 0.1, out=q), want)


# -------------------------------------------------------------------- prompt


def run_prefill(ops, n, first, Hq, H, D, seed, spread=3, q_size=1.0, scale=0.1, rows=None, width=0):
    """A prompt of n tokens behind `first`, checked at `rows` (all by default)."""
    rng = np.random.default_rng(seed)
    q, kc, ke, vc, ve, table = attn_case(rng, [first + n], Hq, H, D, spread, 1.0)
    q = torch.from_numpy((rng.standard_normal((n, Hq, D)) * q_size).astype(np.float32)).bfloat16()
    table = np.concatenate([table[0], np.full(width, -1, dtype=np.int32)])
    dev = q.to(DEV)
    ws = ops.kv8_attn_prefill_workspace(n, first, Hq, H, D, DEV)
    ws[4:] = 255  # partials hold NaN before the call
    out = ops.kv8_attn_prefill(dev, plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table).to(DEV), first,
                               scale, workspace=ws, out=torch.full_like(dev, float("nan")))
    ops.read_status(ws, "kv8_attn_prefill")
    assert not out.isnan().any()
    rows = range(n) if rows is None else sorted({r for r in rows if 0 <= r < n})
    # a query is the sum of two e4m3 numbers of a row whose top is above 224: off by half a step of 2^-9 at most
    check_attn(out[list(rows)], q[list(rows)], kc, ke, vc, ve, [table] * len(rows), [first + r + 1 for r in rows], scale, 2.0 ** -10 / 224)


@pytest.mark.parametrize("Hq,H,D", [(32, 4, 128), (64, 4, 128), (8, 2, 64), (16, 2, 64), (3, 3, 128), (14, 2, 64), (5, 1, 128), (100, 1, 64), (128, 1, 128)])
@pytest.mark.parametrize("n,first", [(1, 0), (1, 300), (17, 0), (50, 78), (33, 1000), (130, 127)])
def test_prefill_heads(ops, Hq, H, D, n, first):
    run_prefill(ops, n, first, Hq, H, D, seed=n + first, rows=[0, 1, 2, 15, 16, 31, 32, 49, n // 2, n - 2, n - 1])


@pytest.mark.parametrize("Hq,H,D", [(8, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("n,first", [(300, 0), (257, 5), (128, 128)])
def test_prefill_every_row(ops, Hq, H, D, n, first):
    run_prefill(ops, n, first, Hq, H, D, seed=n, width=5)


@pytest.mark.parametrize("Hq,H,D,n,first", [(32, 4, 128, 1500, 100), (32, 4, 128, 2048, 0), (8, 8, 128, 700, 900), (16, 2, 64, 2000, 3000), (64, 4, 128, 40, 9001),
                                            (8, 2, 64, 3, 12000), (16, 4, 128, 20000, 0), (128, 1, 64, 700, 5)])
def test_prefill_long(ops, Hq, H, D, n, first):
    run_prefill(ops, n, first, Hq, H, D, seed=n, rows=[0, 1, 127, 128, n // 3, n // 2, n - 17, n - 1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread,q_size,scale", [(0, 1.0, 0.1), (20, 1.0, 0.1), (3, 30.0, 1.0), (3, 1e-30, 1.0), (3, 1e20, 1e-20), (25, 1e-6, 1.0)])
def test_prefill_magnitudes(ops, D, spread, q_size, scale):
    for n, first in ((40, 500), (300, 0)):
        run_prefill(ops, n, first, 8, 2, D, seed=31, spread=spread, q_size=q_size, scale=scale, rows=range(0, n, 7))


def test_prefill_findings_and_refusals(ops):
    rng = np.random.default_rng(32)
    q, kc, ke, vc, ve, table = attn_case(rng, [100], 8, 2, 64)
    args = [plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve)]
    q = torch.zeros(50, 8, 64, device=DEV, dtype=torch.bfloat16)
    err = pkg("_lib").B200Error
    for bad in (-1, kc.shape[0]):
        t = torch.from_numpy(table[0].copy()).to(DEV)
        t[2] = bad
        ws = ops.kv8_attn_prefill_workspace(50, 50, 8, 2, 64, DEV)
        ops.kv8_attn_prefill(q, *args, t, 50, 0.1, workspace=ws)
        with pytest.raises(err, match="pool"):
            ops.read_status(ws, "prefill")
    row = torch.from_numpy(table[0]).to(DEV)
    with pytest.raises(err, match="do not fit"):
        ops.kv8_attn_prefill(q, *args, row, 16 * row.numel() - 49, 0.1)
    with pytest.raises(err, match="workspace"):
        ops.kv8_attn_prefill(q, *args, row, 50, 0.1, workspace=torch.zeros(128, dtype=torch.uint8, device=DEV))
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(table_row=row[None]), dict(table_row=row.long()), dict(out=q[:3]), dict(workspace=row)):
        with pytest.raises(ValueError):
            ops.kv8_attn_prefill(**(dict(q=q, k_pool=args[0], v_pool=args[1], k_scale=args[2], v_scale=args[3], table_row=row, first_pos=0, scale=0.1) | bad))
    assert ops.kv8_attn_prefill(q[:0], *args, row, 50, 0.1).shape == (0, 8, 64)


def test_prefill_nan_reaches_its_key_tile_and_later_rows(ops):
    """A NaN key is masked ahead of its token; a NaN value reaches the rows from at most 127 tokens before it on, in its kv head and column."""
    rng = np.random.default_rng(34)
    n = 400
    q, kc, ke, vc, ve, table = attn_case(rng, [n], 8, 2, 64)
    q = torch.from_numpy(rng.standard_normal((n, 8, 64)).astype(np.float32)).bfloat16().to(DEV)
    args = lambda k, v: (plain.pool_of(k), plain.pool_of(v), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table[0]).to(DEV), 0, 0.1)
    bad = kc.copy()
    bad[table[0, 300 // 16], 1, 300 % 16, 9] = 127
    got = ops.kv8_attn_prefill(q, *args(bad, vc)).isnan()
    assert not got[:, :4].any() and not got[:300].any() and got[300:, 4:].all()
    bad = vc.copy()
    bad[table[0, 300 // 16], 0, 300 % 16, 9] = 255
    got = ops.kv8_attn_prefill(q, *args(kc, bad)).isnan()
    assert not got[:, 4:].any() and not got[:300 - 127].any() and got[300:, :4, 9].all()
    got[:, :4, 9] = False
    assert not got.any()
    bad = q.clone()
    bad[7, 3, 2] = float("inf")
    bad[200, 5, 60] = float("nan")
    got = ops.kv8_attn_prefill(bad, *args(kc, vc)).isnan()
    assert got[7, 3].all() and got[200, 5].all() and int(got.sum()) == 128


def test_prefill_captured_on_another_stream_beside_a_second_call(ops):
    """A captured prompt pass - append, then attention over keys shared out in parts - replayed with other rows in its buffers, while a
    call with a workspace of its own runs on a second stream."""
    rng = np.random.default_rng(35)
    H, Hq, D, n, first = 2, 8, 128, 40, 3000
    _, kc, ke, vc, ve, table = attn_case(rng, [first + n], Hq, H, D)
    codes = [np.where(c & 127 == 127, 0, c) for c in (kc, vc)]
    cache = [plain.pool_of(c.copy()) for c in codes] + [plain.scale_of(ke), plain.scale_of(ve)]
    other = [c.clone() for c in cache]
    row = torch.from_numpy(table[0]).to(DEV)
    slots = ints([int(table[0, p // 16]) * 16 + p % 16 for p in range(first, first + n)])
    q = torch.zeros(n, Hq, D, device=DEV, dtype=torch.bfloat16)
    k, v = torch.zeros(n, H, D, device=DEV, dtype=torch.bfloat16), torch.zeros(n, H, D, device=DEV, dtype=torch.bfloat16)
    ws = [ops.kv8_attn_prefill_workspace(n, first, Hq, H, D, DEV) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        ops.kv8_append(k, v, *cache, slots)
        out = ops.kv8_attn_prefill(q, *cache, row, first, 0.1, workspace=ws[0])
    still = torch.randn(n, Hq, D, device=DEV).bfloat16()
    with torch.cuda.stream(streams[1]):
        alone = ops.kv8_attn_prefill(still, *other, row, first, 0.1, workspace=ws[1])
    host = [c.copy() for c in codes], [ke.copy(), ve.copy()]
    for turn in range(3):
        rows = rows_of(rng, n, H, D, torch.bfloat16)
        with torch.cuda.stream(streams[0]):
            q.copy_(torch.from_numpy(rng.standard_normal((n, Hq, D)).astype(np.float32)))
            for x, r in zip((k, v), rows):
                x.copy_(torch.from_numpy(r))
            torch.cuda.synchronize()
            graph.replay()
        with torch.cuda.stream(streams[1]):
            again = [ops.kv8_attn_prefill(still, *other, row, first, 0.1, workspace=ws[1]) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, alone) for a in again)
        for x, c, e in zip((k, v), *host):
            plain.append(x.double().cpu().numpy(), slots.tolist(), c, e)
        check_attn(out, q.cpu(), host[0][0], host[1][0], host[0][1], host[1][1], [table[0]] * n, range(first + 1, first + n + 1), 0.1, 2.0 ** -10 / 224)


def test_prefill_agrees_with_decode(ops):
    """The last row of a prompt is a decode row."""
    rng = np.random.default_rng(33)
    _, kc, ke, vc, ve, table = attn_case(rng, [777], 32, 4, 128)
    args = [plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve)]
    q = torch.randn(20, 32, 128, device=DEV).bfloat16()
    t = torch.from_numpy(table).to(DEV)
    a = ops.kv8_attn_prefill(q, *args, t[0], 757, 0.09)[19].float()
    b = ops.kv8_attn_decode(q[19:].contiguous(), *args, t, ints([777]), 0.09)[0].float()
    # both within half a bf16 step and 2^-11 of weights of the exact value
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -9 * b.abs().max()).all()


# --------------------------------------------------------------- used together


@pytest.mark.parametrize("Hq,H,D,dtype", [(32, 4, 128, torch.bfloat16), (8, 2, 64, torch.float32)])
def test_prompts_then_decode_steps(ops, Hq, H, D, dtype):
    """Three sequences: prompts into the cache, then 20 decode steps, as one captured step that is replayed on another stream.  Pages come
    from the free list on the GPU; every step's attention equals the 64-bit one over a cache kept by the plain restatement."""
    rng = np.random.default_rng(21)
    prompts, width, blocks = [37, 1, 16], 6, 24
    B = len(prompts)
    cache = ops.kv8_pools(blocks, H, D, DEV)
    supply = ints([int(i) for i in rng.permutation(blocks)])
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    status = status_word()
    host = [np.zeros((blocks, H, 16, D), dtype=np.uint8) for _ in range(2)], [np.full((blocks, H), -32) for _ in range(2)]

    def host_append(k, v, slots):
        for x, codes, exps in zip((k, v), *host):
            plain.append(x.double().cpu().numpy(), slots.tolist(), codes, exps)

    k, v = (torch.from_numpy(r).to(DEV, dtype) for r in rows_of(rng, 64, H, D, dtype))
    m = ops.kv_slot_map(ints([0] * B), ints(prompts), table, supply, ints([0]), 64, blocks, status=status)
    ops.kv8_append(k, v, *cache, m.slots, status=status)
    host_append(k, v, m.slots)

    one, used, ctx = ints([1] * B), m.supply_used.clone(), m.lens.clone()
    q = torch.zeros(B, Hq, D, device=DEV, dtype=torch.bfloat16)
    k, v = torch.zeros(B, H, D, device=DEV, dtype=dtype), torch.zeros(B, H, D, device=DEV, dtype=dtype)
    ws = ops.kv8_attn_workspace(B, Hq, H, D, width, DEV)

    def step():
        m = ops.kv_slot_map(ctx, one, table, supply, used, B, blocks, status=status)
        ops.kv8_append(k, v, *cache, m.slots, status=status)
        out = ops.kv8_attn_decode(q, *cache, table, m.lens, D ** -0.5, workspace=ws)
        ctx.copy_(m.lens)
        used.copy_(m.supply_used)
        return m.slots, out

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):  # the first launches of these kernels in the process may be in here
        slots, out = step()
    with torch.cuda.stream(stream):
        for i in range(20):
            q.copy_(torch.from_numpy(rng.standard_normal((B, Hq, D)).astype(np.float32)))
            for x, r in zip((k, v), rows_of(rng, B, H, D, dtype)):
                x.copy_(torch.from_numpy(r))
            graph.replay()
            stream.synchronize()
            host_append(k, v, slots)
            lens = [p + i + 1 for p in prompts]
            assert ctx.tolist() == lens
            check_attn(out, q.cpu(), host[0][0], host[1][0], host[0][1], host[1][1], table.cpu().numpy(), lens, D ** -0.5)
    for pool, codes in zip(cache[:2], host[0]):
        assert np.array_equal(pool.view(torch.uint8).cpu().numpy(), codes)
    ops.read_status(status, "steps")
    ops.read_status(ws, "attention")


def test_two_calls_at_once_and_again(ops):
    """Two streams with a workspace each give what the calls give alone, bit for bit."""
    rng = np.random.default_rng(22)
    lens = [900, 33, 0, 2000]
    case = attn_case(rng, lens, 16, 2, 64)
    q, kc, ke, vc, ve, table = case
    args = [q.to(DEV), plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table).to(DEV)]
    lens_dev = [ints(lens), ints([min(a, b) for a, b in zip(lens, lens[::-1])])]
    alone = [ops.kv8_attn_decode(*args, n, 0.1) for n in lens_dev]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [ops.kv8_attn_workspace(4, 16, 2, 64, table.shape[1], DEV) for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.kv8_attn_decode(*args, lens_dev[i], 0.1, workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


@pytest.mark.parametrize("Hq,H,D", [(32, 4, 128), (64, 4, 128), (16, 2, 64), (7, 1, 128), (40, 1, 128), (16, 8, 64), (64, 8, 128)])
@pytest.mark.parametrize("lens", [[1, 40, 531, 16], [9000], [700] * 40])
def test_decode_query_heads_that_are_not_finite(ops, Hq, H, D, lens):
    """A NaN or an infinity in the query of one head of each group: that head is NaN, all others have their own weights.  (Their bits may change: the
    heads of a group move their references together, and a weight below 2^-14 is rounded to the reference's steps, which the tolerance counts.)"""
    rng = np.random.default_rng(40)
    q, kc, ke, vc, ve, table = attn_case(rng, lens, Hq, H, D)
    clean = run_decode(ops, q, kc, ke, vc, ve, table, lens, 0.1)
    hit = torch.zeros(len(lens), Hq, dtype=torch.bool)
    bad = q.clone()
    for b in range(len(lens)):
        for g in range(H):
            h = g * (Hq // H) + int(rng.integers(Hq // H))
            bad[b, h, int(rng.integers(D))] = [float("nan"), float("inf"), -float("inf")][(b + g) % 3]
            hit[b, h] = True
    got = run_decode(ops, bad, kc, ke, vc, ve, table, lens, 0.1).cpu()
    assert got[hit].isnan().all()
    got[hit] = clean.cpu()[hit]
    check_attn(got, q, kc, ke, vc, ve, table, lens, 0.1)


@pytest.mark.parametrize("Hq,H,D", [(32, 4, 128), (64, 4, 128), (16, 2, 64), (40, 1, 128)])
def test_decode_query_heads_far_apart(ops, Hq, H, D):
    """Heads of one kv head whose queries differ by up to 2^120 each have their own weights."""
    rng = np.random.default_rng(41)
    lens = [100, 1, 700]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, Hq, H, D)
    q = (q.double() * 2.0 ** torch.tensor([0, 60, -60, 0, 15, -15, 30])[torch.arange(Hq) % 7][:, None]).bfloat16()
    check_attn(run_decode(ops, q, kc, ke, vc, ve, table, lens, 0.1), q, kc, ke, vc, ve, table, lens, 0.1)


def test_slot_map_pages_that_cannot_be_had(ops):
    """Rows of a table that was used before hold ids of pages that are others' by now: where no page, or none that is one, can be handed out, the entry says so."""
    was = np.arange(100, 100 + 4 * 5, dtype=np.int32).reshape(4, 5)
    for supply, used, gets, code in (([7, 8], 0, [7, 8, -1, -1], 21), ([7, 8], 2, [-1] * 4, 21), ([7, 8], 3, [-1] * 4, 21), ([7, 8], -1, [-1] * 4, 21),
                                     ([], 0, [-1] * 4, 21), ([7, 999, -3, 8], 0, [7, -1, -1, 8], 16)):
        table, status = torch.from_numpy(was.copy()).to(DEV), status_word()
        m = ops.kv_slot_map(ints([16, 3, 0, 20]), ints([33, 2, 1, 1]), table, ints(supply), ints([used]), 40, 200, status=status)
        want = was.copy()
        want[0, 1:4], want[2, 0] = gets[:3], gets[3]
        assert table.tolist() == want.tolist() and status.item() == code
        assert m.lens.tolist() == [49, 5, 1, 21] and m.row_start.tolist() == [0, 33, 35, 36, 37]
        slots = [want[0, 1 + i // 16] * 16 + i % 16 if want[0, 1 + i // 16] >= 0 else -1 for i in range(33)] + [105 * 16 + 3, 105 * 16 + 4]
        assert m.slots.tolist() == slots + [want[2, 0] * 16 if want[2, 0] >= 0 else -1, 116 * 16 + 4] + [-1] * 3


def test_a_step_after_pages_ran_out_touches_no_page_of_others(ops):
    """Sequence 0 needs a page that is not there, and its table row still names one from before, sequence 1's.  The steps after that go on with the lengths."""
    rng = np.random.default_rng(42)
    H, D, blocks = 2, 64, 8
    codes, exps = plain.random_cache(rng, blocks, H, D)
    cache = [plain.pool_of(codes.copy()), plain.pool_of(codes.copy()), plain.scale_of(exps), plain.scale_of(exps)]
    table, ctx, used = ints([[1, 3, 3], [2, 3, -1]]), ints([15, 20]), ints([1])
    for step in range(3):
        status = status_word()
        m = ops.kv_slot_map(ctx, ints([1, 0]), table, ints([5]), used, 1, blocks, status=status)
        k, v = (torch.from_numpy(r).to(DEV) for r in rows_of(rng, 1, H, D, torch.float32))
        ops.kv8_append(k, v, *cache, m.slots, status=status)
        assert status.item() == [0, 21, 16][step] and m.slots.tolist() == [[31], [-1], [-1]][step]
        ctx, used = m.lens, m.supply_used
    for pool in cache[:2]:
        got = pool.view(torch.uint8).cpu().numpy()
        assert np.array_equal(np.delete(got, 1, 0), np.delete(codes, 1, 0))
    assert table.tolist() == [[1, -1, 3], [2, 3, -1]]


@pytest.mark.parametrize("H,D", [(1, 64), (1, 128), (100, 64), (100, 128)])
def test_prefill_value_of_nan_whose_weight_vanishes(ops, H, D):
    """A NaN value under a weight of 2^-400: a softmax in floating point multiplies it by zero, which is NaN."""
    rng = np.random.default_rng(45)
    n, first = 2, 254
    _, kc, ke, vc, ve, table = attn_case(rng, [first + n], H, H, D)
    ke[:], ve[:] = 0, 0
    kc[:] = 0
    q = torch.ones(n, H, D, device=DEV, dtype=torch.bfloat16)
    for t in range(128, 256):  # the second tile of keys: scores of 8 D
        kc[table[0, t // 16], :, t % 16] = int(plain.encode(np.array([8.0]))[0])
    vc[table[0, 0], 0, 3, 5] = 127
    got = ops.kv8_attn_prefill(q, plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve), ints(table[0].tolist()), first, 1.0).isnan()
    assert got[:, 0, 5].all() and int(got.sum()) == n


def prompt_of(ops, n, first, Hq, H, D, seed):
    rng = np.random.default_rng(seed)
    _, kc, ke, vc, ve, table = attn_case(rng, [first + n], Hq, H, D)
    q = torch.from_numpy(rng.standard_normal((n, Hq, D)).astype(np.float32)).bfloat16().to(DEV)

    def run(v, k=kc):
        ws = ops.kv8_attn_prefill_workspace(n, first, Hq, H, D, DEV)
        ws[4:] = 255
        out = ops.kv8_attn_prefill(q, plain.pool_of(k), plain.pool_of(v), plain.scale_of(ke), plain.scale_of(ve), torch.from_numpy(table[0]).to(DEV), first, 0.1,
                                   workspace=ws, out=torch.full_like(q, float("nan")))
        ops.read_status(ws, "prompt")
        return out

    return run, kc, vc, table[0]


@pytest.mark.parametrize("Hq,H,D,n,first", [(32, 32, 64, 2048, 1), (32, 32, 128, 700, 1), (32, 4, 128, 1500, 77), (8, 2, 64, 400, 0), (3, 3, 128, 130, 5), (64, 4, 128, 17, 5001),
                                            (8, 2, 128, 300, 900), (5, 1, 64, 200, 333), (100, 1, 64, 9, 120), (4, 4, 64, 128, 127)])
def test_prefill_masked_values_of_nan_reach_nothing(ops, Hq, H, D, n, first):
    """A NaN value of a token is NaN in its column for the rows from that token on and nothing to the rows ahead of it, which keep their bits."""
    run, _, vc, row = prompt_of(ops, n, first, Hq, H, D, seed=43)
    clean, bad = run(vc), vc.copy()
    rng = np.random.default_rng(44)
    want = torch.zeros(n, Hq, D, dtype=torch.bool)
    last = first + n - 1
    for t in {0, first, first + 1, first + n // 2, (first + n // 2) // 128 * 128 + 127, first + min(n - 1, 255), last - 1, last, *(int(x) for x in rng.integers(first, first + n, 4))}:
        if not 0 <= t <= last:
            continue
        h, c = int(rng.integers(H)), int(rng.integers(D))
        bad[row[t // 16], h, t % 16, c] = (127, 255)[t & 1]
        want[max(t - first, 0):, h * (Hq // H):(h + 1) * (Hq // H), c] = True
    got = run(bad)
    assert torch.equal(got.isnan().cpu(), want)
    assert torch.equal(got.cpu()[~want], clean.cpu()[~want])


def test_status_words_off_their_boundary_are_refused(ops):
    odd = torch.zeros(12, dtype=torch.uint8, device=DEV)[2:10]
    pools = ops.kv8_pools(4, 2, 64, DEV)
    x, slots = torch.zeros(3, 2, 64, device=DEV), ints([0, 1, 2])
    with pytest.raises(pkg("_lib").B200Error, match="4-byte"):
        ops.kv8_append(x, x, *pools, slots, status=odd)
    with pytest.raises(pkg("_lib").B200Error, match="4-byte"):
        ops.kv_slot_map(slots, slots, slots.view(3, 1), slots, slots[:1], 4, 4, status=odd)


def test_findings_without_a_workspace(ops):
    rng = np.random.default_rng(46)
    lens = [40, 40]
    q, kc, ke, vc, ve, table = attn_case(rng, lens, 8, 2, 64)
    cache = [plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve)]
    q, good = q.to(DEV), torch.from_numpy(np.where(table < 0, 0, table)).to(DEV)
    bad = good.clone()
    bad[1, 1] = 10 ** 6
    for call in (lambda t, s: ops.kv8_attn_decode(q, *cache, t, ints(lens), 0.1, status=s), lambda t, s: ops.kv8_attn_prefill(q, *cache, t[1], 38, 0.1, status=s)):
        status = status_word()
        want = call(good, status)
        assert status.item() == 0 and torch.equal(want, call(good, None))
        call(bad, status)
        assert status.item() == 16


def test_status_beside_a_workspace_is_refused(ops):
    pools = ops.kv8_pools(4, 2, 64, DEV)
    q, table, lens = torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16), ints([[0], [1], [2]]), ints([1, 2, 3])
    ws = ops.kv8_attn_workspace(3, 4, 2, 64, 1, DEV)
    for bad in (dict(status=status_word(), workspace=ws), dict(status=torch.zeros(1, dtype=torch.int32)), dict(status=torch.zeros(3, dtype=torch.uint8, device=DEV))):
        with pytest.raises(ValueError, match="status"):
            ops.kv8_attn_decode(q, *pools, table, lens, 0.1, **bad)
        with pytest.raises(ValueError, match="status"):
            ops.kv8_attn_prefill(q, *pools, table[0], 0, 0.1, **bad)


def test_findings_without_a_workspace_in_a_captured_call(ops):
    """The first finding stays: a later clean call leaves it in the status word."""
    rng = np.random.default_rng(49)
    q, kc, ke, vc, ve, table = attn_case(rng, [40, 40], 8, 2, 64)
    cache = [plain.pool_of(kc), plain.pool_of(vc), plain.scale_of(ke), plain.scale_of(ve)]
    q, table, status = q.to(DEV), torch.from_numpy(np.where(table < 0, 0, table)).to(DEV), status_word()
    want = ops.kv8_attn_decode(q, *cache, table, ints([40, 40]), 0.1)
    lens = ints([40, 40])
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = ops.kv8_attn_decode(q, *cache, table, lens, 0.1, status=status)
    codes = []
    with torch.cuda.stream(stream):
        for L in (40, -1, 40):
            lens.fill_(L)
            graph.replay()
            stream.synchronize()
            codes.append(status.item())
    assert codes == [0, 17, 17] and torch.equal(out, want)
