"""What the page pool, the normed append, the windowed attention and the adjusted logits launch for a call's shapes.  No
GPU."""
import ctypes

import pytest

from launches import Recorder
from test_gpu_norm_append import MANY
from test_gpu_window import CASES, CROWDS, DEALT, TILES
from test_serve_host import batch, cache
from test_step_host import pool, rules

A = ctypes.addressof
T = {"f32": 0, "f16": 1, "bf16": 2}


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    return Recorder(str(tmp_path_factory.mktemp("launches")))


def window(launched, args, win, decode=False):
    new, lens, P, H, HKV, D, q, kv, page, hf, pad = args
    n, rows = sum(new) + pad, max(-(-x // page) for x in lens + [1])
    c = cache(type=T[kv], n_pages=1000, page_size=page, n_kv_heads=HKV, head_dim=D, page_stride=HKV * page * D,
              row_stride=D if hf else HKV * D, head_stride=page * D if hf else D)
    b = batch(table_stride=rows, table_width=rows, n_seqs=len(lens), n_tokens=n, q_start=None if decode else 0x8000,
              prefix=0x9000 if P else None, prefix_len=P)
    need = launched.lib.bpd_attn_window_paged_workspace(A(c), A(b), T[q], H, *win)
    got = launched("bpd_attn_window_paged_gpu", A(c), A(b), 1 << 30, H * D, 1 << 40, H * D, None, T[q], H, 0.1, *win,
                   0x50000 if need else None, need)
    return need, got


@pytest.mark.parametrize("case", range(len(TILES)))
def test_tiles_are_planned(launched, case):
    need, got = window(launched, *TILES[case])
    assert [l.kernel for l in got] == ["k_attn_plan", "k_attn_tile", "k_attn_join"] and need > 0


@pytest.mark.parametrize("case", range(len(DEALT)))
def test_long_windows_of_few_sequences_are_dealt(launched, case):
    need, got = window(launched, *DEALT[case], decode=True)
    assert [l.kernel for l in got] == ["k_attn_wave", "k_attn_join"] and need > 0


@pytest.mark.parametrize("case", range(len(CASES)))
def test_small_batches_take_one_launch_and_no_workspace(launched, case):
    args, win = CASES[case]
    need, got = window(launched, args, win)
    assert [l.kernel for l in got] == ["k_attn_head"] and need == 0
    new, H, HKV = args[0], args[3], args[4]
    tiles = sum(-(-n * (H // HKV) // 16) for n in new)
    assert got[0].grid[0] % HKV == 0 and got[0].grid[0] // HKV >= tiles and got[0].block[0] in (256, 512)


def test_a_workgroup_for_each_sequence_and_head(launched):
    for B, HKV, D in ((1, 8, 64), (64, 8, 128), (300, 2, 256)):
        _, (one,) = window(launched, ([1] * B, [600] * B, 0, 4 * HKV, HKV, D, "bf16", "bf16", 64, True, 0), (512, 4), decode=True)
        assert one.kernel == "k_attn_head" and one.grid[0] == B * HKV
        assert one.block[0] == (256 if D == 256 or B * HKV > 256 else 512)


@pytest.mark.parametrize("case", range(len(CROWDS)))
def test_waves_of_many_sequences(launched, case):
    args, win, waves = CROWDS[case]
    need, (one,) = window(launched, args, win, decode=max(args[0]) == 1)
    assert one.kernel == "k_attn_head" and need == 0 and one.block[0] == 64 * waves


def test_slices_of_logits(launched):
    for B, V in ((1, 7), (1, 32000), (64, 128256), (4000, 1000), (1, 1 << 22), (255, 1 << 22)):
        r = rules(mask_stride=1 << 20)
        (one,) = launched("bpd_adjust_logits_gpu", 1 << 40, 0, V, 1 << 50, 0, V, B, V, A(r))
        assert one.kernel == "k_adjust" and one.grid[0] % B == 0 and one.lds == 0
        S = one.grid[0] // B
        assert any(S == -(-V // n) for n in (1024, 2048, 4096, 8192)) and one.grid[0] < 1 << 31


def test_the_pool_takes_one_launch_a_call(launched):
    for B, W, n in ((1, 5, 100000), (256, 513, 1024), (16384, 9, 20000)):
        p = pool(n_rows=max(B, 300), table_width=W, table_stride=W, n_pages=1000)
        (one,) = launched("bpd_pages_extend_gpu", A(p), 0x6000, 0x7000, B, n, 0, 0x8000, W, 0x9000, 0xA000, 0xB000, 0xC000, 0xD000)
        (two,) = launched("bpd_pages_release_gpu", A(p), 0x6000, 0x7000, B, 0, 0)
        for l in (one, two):
            assert 1 <= l.grid[0] <= 1024 and l.lds == 4 * max(B, 300)
        assert (one.kernel, two.kernel) == ("k_extend", "k_release")


def test_waves_of_a_token(launched):
    c = cache(n_kv_heads=8, head_dim=128, page_stride=16 * 8 * 128, row_stride=128, head_stride=16 * 128)
    for n, H, waves in ((1, 32, 4), (1024, 32, 4), (1025, 32, 2), (5000, 4, 2)):
        b = batch(n_seqs=n, n_tokens=n)
        (one,) = launched("bpd_norm_rope_append_paged_gpu", A(c), A(b), 0x80000, 0, 0x90000, 0, 0, 1e-6, None, None, 1 << 40,
                          H * 128, 1 << 41, 1024, 1 << 42, 1024, 1 << 43, H * 128, 1, H)
        assert one.kernel == "k_norm_append" and one.grid[0] == n and one.block[0] == 64 * waves


@pytest.mark.parametrize("case,waves", [(0, 2), (1, 2), (2, 1)])
def test_waves_of_many_tokens(launched, case, waves):
    new, lens, P, H, HKV, D, x, kv, page, hf, pad, rot, neox, w = MANY[case]
    n = sum(new) + pad
    c = cache(type=T[kv], page_size=page, n_kv_heads=HKV, head_dim=D, page_stride=page * HKV * D, row_stride=D,
              head_stride=page * D)
    b = batch(n_seqs=2, n_tokens=n, q_start=0x8000)
    (one,) = launched("bpd_norm_rope_append_paged_gpu", A(c), A(b), 0x80000, 0, 0x90000, 0, T[w], 1e-6, None, None, 1 << 40,
                      H * D, 1 << 41, HKV * D, 1 << 42, HKV * D, 1 << 43, H * D, T[x], H)
    assert one.kernel == "k_norm_append" and one.block[0] == 64 * waves
