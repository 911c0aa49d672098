"""CPU models of the index arithmetic in the row kernels: every column of a row belongs
to one thread, copies and table entries stay within their arrays, the column sums'
workspace is as large as any launch."""
import math

import pytest
import torch

FWD = {2: [(256, 32, 1), (512, 32, 2), (1024, 32, 4), (2048, 64, 4), (4096, 128, 4), (8192, 256, 4)],
       4: [(256, 32, 1), (512, 32, 2), (1024, 64, 2), (2048, 128, 2), (4096, 256, 2), (8192, 512, 2)]}
BWD = {2: [(256, 32, 1), (512, 32, 2), (1024, 64, 2), (2048, 128, 2), (4096, 256, 2), (8192, 512, 2)],
       4: [(256, 32, 1), (512, 32, 2), (1024, 128, 1), (2048, 256, 1), (4096, 512, 1), (8192, 512, 2)]}
WIDTHS = [1, 7, 8, 250, 256, 264, 504, 512, 513, 1000, 1024, 1032, 2048, 2050, 4088, 4096, 4104, 8184, 8191, 8192]


def shape(table, size, cols):
    return next((nt, nv) for most, nt, nv in table[size] if cols <= most)


def columns(nt, nv, size, vectors):
    """Column of (thread, group, value) in a kernel's tile."""
    tid = torch.arange(nt)[:, None, None]
    g = torch.arange(nv)[None, :, None]
    i = torch.arange(8)[None, None, :]
    if not vectors:
        return (g * 8 + i) * nt + tid
    per = 16 // size
    return ((g * (8 // per) + i // per) * nt + tid) * per + i % per


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("table", [FWD, BWD], ids=["forward", "gradient"])
def test_every_column_has_one_thread(table, size):
    for cols in WIDTHS:
        nt, nv = shape(table, size, cols)
        assert cols <= nt * nv * 8
        for vectors in ([True, False] if cols % 8 == 0 else [False]):
            c = columns(nt, nv, size, vectors)
            assert torch.equal(c.flatten().sort().values, torch.arange(nt * nv * 8))
            if vectors:  # a piece of 16 bytes lies within the width or past it
                first = c[:, :, ::16 // size]
                assert bool(((first < cols) == (first + 16 // size <= cols)).all())


@pytest.mark.parametrize("size", [2, 4])
def test_staged_rows_fit_their_region(size):
    """Rows that start anywhere: the 16-byte pieces that cover a row, and what is read of them."""
    for cols in WIDTHS:
        region = ((cols * size + 15) // 16 + 1) * 16
        for start in range(0, 32, size):
            at, off = start // 16 * 16, start % 16
            pieces = (start + cols * size - at + 15) // 16
            assert pieces * 16 <= region and off + cols * size <= pieces * 16


def test_workspace_holds_every_launch():
    for cols in WIDTHS:
        nt = 32 if cols <= 512 else 64 if cols <= 1024 else 128 if cols <= 2048 else 256 if cols <= 4096 else 512
        for size in (2, 4):
            threads = shape(BWD, size, cols)[0]
            for rows in (1, 100, 148, 700, 5000, 10 ** 6):
                have = min(rows, 148 * (512 // nt))
                for few in (2, 4):
                    assert min(rows, 148 * (512 // threads), max(rows // few, 148)) <= have


def test_gelu_table_entries():
    """A code's FP16 bits and its group's unit name the entry of its own value."""
    pad, half, end, low = 48, 256, 64, -24
    codes = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn)
    bits = codes.to(torch.float16).view(torch.int16).to(torch.int64) & 0xFFFF
    for byte in range(112, 127):  # the units in the window
        e = byte - 127
        entry = 8 * (e + 9) + (bits >> 7)
        assert int((pad + entry).min()) >= 0 and int((pad + entry).max()) < pad + 2 * half + end
        for code, at in zip(codes.float().tolist(), entry.tolist()):
            if code == 0.0 or math.isnan(code):
                continue
            k = at - half if code < 0 else at
            assert 0 <= k < half
            value = 2.0 ** (low + k // 8) * (1 + k % 8 / 8)
            assert value == abs(code) * 2.0 ** e


def test_parts_of_a_clusters_row_cover_it():
    for vocab in (8192, 8193, 20001, 32003, 50304):
        for C in (1, 2, 4):
            for per in (4, 8):
                chunk = vocab if C == 1 else ((vocab + C - 1) // C + per - 1) // per * per
                ends = [(min(vocab, r * chunk), min(vocab, min(vocab, r * chunk) + chunk)) for r in range(C)]
                assert ends[0][0] == 0 and ends[-1][1] == vocab
                assert all(a[1] == b[0] for a, b in zip(ends, ends[1:]))
