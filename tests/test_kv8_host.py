"""The 8-bit page cache without a GPU: its plain restatement, and the refusals of its entry points."""
import numpy as np
import pytest
import torch

import kv8_cases as plain
from conftest import pkg

P = 4096  # an address that no kernel sees: every call here is refused first


def refused(rc: int, *words: str) -> None:
    assert rc == -1
    detail = pkg("_lib").load().b200_last_error_detail().decode()
    assert all(w in detail for w in words), detail


def test_encode_is_the_e4m3_rounding_of_torch():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 2.0 ** rng.integers(-12, 9, 20000), plain.CODES, (plain.CODES[1:] + plain.CODES[:-1]) / 2,
                        [448.0, 440.0, 2.0 ** -10, 2.0 ** -11, 0.0, -0.0]])
    x = x[np.abs(x) <= 448]
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(plain.E4M3).view(torch.uint8).numpy()
    assert np.array_equal(plain.encode(x.astype(np.float64)), want)
    assert list(plain.encode(np.array([1e9, -1e9, np.inf, -np.inf, np.nan]))) == [126, 254, 127, 127, 127]


@pytest.mark.parametrize("top,e", [(0.0, -32), (448.0, 0), (448.0001, 1), (224.0, -1), (1.75, -8), (1.7500001, -7), (2.0 ** -60, -32), (1e30, 31)])
def test_fit(top, e):
    assert plain.fit(top) == e


def test_append_refuses():
    lib = pkg("_lib").load()

    def call(kn=P, vn=P, ks=512, vs=512, kp=P, vp=P, kc=P, vc=P, slots=P, rows=4, heads=4, dim=128, blocks=9, dtype=0):
        return lib.b200_kv8_append(kn, vn, ks, vs, kp, vp, kc, vc, slots, None, rows, heads, dim, blocks, dtype, None)

    for name in ("kn", "vn", "kp", "vp", "kc", "vc", "slots"):
        refused(call(**{name: None}), "null")
    refused(call(rows=0), "non-positive")
    refused(call(heads=0), "non-positive")
    refused(call(blocks=-1), "non-positive")
    refused(call(dim=96), "head_dim 96")
    refused(call(dtype=2), "dtype 2")
    refused(call(blocks=2 ** 27), "32 bits")
    refused(call(kn=P + 8), "multiples of 16")
    refused(call(dtype=1, vs=514), "multiples of 16")
    refused(call(ks=-512), "multiples")
    refused(call(vp=P + 8), "16-byte aligned")


def test_slot_map_refuses():
    lib = pkg("_lib").load()

    def call(ctx=P, new=P, table=P, supply=P, used=P, n=5, lens=P + 64, start=P, seq=P, pos=P, slots=P, out=P + 128, B=3, rows=7, blocks=9, width=4):
        return lib.b200_kv_slot_map(ctx, new, table, supply, used, n, lens, start, seq, pos, slots, out, None, B, rows, blocks, width, None)

    for name in ("ctx", "new", "table", "supply", "used", "lens", "start", "seq", "pos", "slots", "out"):
        refused(call(**{name: None}), "null")
    refused(call(B=0), "sequences")
    refused(call(B=4097), "4096")
    refused(call(rows=-1), "dimension")
    refused(call(n=-1), "dimension")
    refused(call(blocks=0), "dimension")
    refused(call(width=0), "dimension")
    refused(call(B=4096, width=2 ** 15), "2^31")
    refused(call(blocks=2 ** 27), "2^31")
    refused(call(lens=P), "an output is an input")
    refused(call(out=P), "an output is an input")


def test_decode_refuses():
    lib = pkg("_lib").load()

    def call(q=P, kp=P, vp=P, ks=P, vs=P, table=P, ctx=P, out=P, ws=P, n=1 << 20, B=2, hq=8, hkv=2, dim=64, blocks=9, width=4, scale=0.1, split=0):
        return lib.b200_kv8_attn_decode(q, kp, vp, ks, vs, table, ctx, out, ws, n, B, hq, hkv, dim, blocks, width, scale, split, None)

    for name in ("q", "kp", "vp", "ks", "vs", "table", "ctx", "out", "ws"):
        refused(call(**{name: None}), "null")
    for name in ("B", "hq", "hkv", "blocks", "width"):
        refused(call(**{name: 0}), "non-positive")
    refused(call(hq=7), "multiple of kv heads")
    refused(call(dim=256), "head_dim 256")
    refused(call(width=2 ** 27), "2^31")
    refused(call(blocks=2 ** 27), "2^31")
    for name in ("q", "kp", "vp", "out"):
        refused(call(**{name: P + 8}), "16-byte")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(call(scale=scale), "scale")
    refused(call(B=2 ** 20, width=2 ** 12), "2^31 entries")
    refused(call(split=24), "split_tokens 24")
    refused(call(split=-16), "split_tokens -16")


def test_prefill_refuses():
    lib = pkg("_lib").load()

    def call(q=P, kp=P, vp=P, ks=P, vs=P, table=P, out=P, ws=P, n=1 << 20, R=5, first=0, hq=8, hkv=2, dim=64, blocks=9, width=4, scale=0.1):
        return lib.b200_kv8_attn_prefill(q, kp, vp, ks, vs, table, out, ws, n, R, first, hq, hkv, dim, blocks, width, scale, None)

    for name in ("q", "kp", "vp", "ks", "vs", "table", "out", "ws"):
        refused(call(**{name: None}), "null")
    for name in ("R", "hq", "hkv", "blocks", "width"):
        refused(call(**{name: 0}), "non-positive")
    refused(call(hq=7), "multiple of kv heads")
    refused(call(hq=258), "128 q heads")
    refused(call(dim=96), "head_dim 96")
    refused(call(first=-1), "positions -1")
    refused(call(first=60), "do not fit 4 pages")
    refused(call(first=2 ** 31 - 2), "do not fit")
    refused(call(first=2 ** 31 - 100, R=50, width=2 ** 27 - 1), "2^31")
    refused(call(scale=-0.1), "scale")
    for name in ("q", "kp", "vp", "out"):
        refused(call(**{name: P + 8}), "16-byte")


def test_wrappers_refuse_what_is_not_on_a_gpu():
    ops = pkg("ops")
    i = torch.zeros(3, dtype=torch.int32)
    pools = ops.kv8_pools(4, 2, 64, device="cpu")
    assert pools[0].dtype == torch.float8_e4m3fn and float(pools[2].float().max()) == 2.0 ** -32
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_slot_map(i, i, i.view(3, 1), i, i[:1], 4, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), *pools, i)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_attn_decode(torch.zeros(3, 4, 64, dtype=torch.bfloat16), *pools, i.view(3, 1), i, 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_attn_prefill(torch.zeros(3, 4, 64, dtype=torch.bfloat16), *pools, i, 0, 0.1)


def test_whole_numbers_and_status_words_off_their_boundary_are_refused():
    """A word that the GPU would read, or record a finding in, has to lie on a multiple of its 4 bytes: an access off it is a fault there."""
    lib = pkg("_lib").load()

    def slot_map(**at):
        a = dict(ctx=P, new=P, table=P, supply=P, used=P, lens=P + 64, start=P, seq=P, pos=P, slots=P, out=P + 128, status=P) | at
        return lib.b200_kv_slot_map(a["ctx"], a["new"], a["table"], a["supply"], a["used"], 5, a["lens"], a["start"], a["seq"], a["pos"], a["slots"], a["out"],
                                    a["status"], 3, 7, 9, 4, None)

    for name in ("ctx", "new", "table", "supply", "used", "lens", "start", "seq", "pos", "slots", "out", "status"):
        for off in (1, 2, 3):
            refused(slot_map(**{name: P + 256 + off}), "4-byte")

    def append(slots=P, status=P):
        return lib.b200_kv8_append(P, P, 512, 512, P, P, P, P, slots, status, 4, 4, 128, 9, 0, None)

    refused(append(slots=P + 2), "4-byte")
    refused(append(status=P + 1), "4-byte")

    def decode(table=P, ctx=P):
        return lib.b200_kv8_attn_decode(P, P, P, P, P, table, ctx, P, P, 1 << 20, 2, 8, 2, 64, 9, 4, 0.1, 0, None)

    refused(decode(table=P + 2), "4-byte")
    refused(decode(ctx=P + 3), "4-byte")
    refused(lib.b200_kv8_attn_prefill(P, P, P, P, P, P + 1, P, P, 1 << 20, 5, 0, 8, 2, 64, 9, 4, 0.1, None), "4-byte")
