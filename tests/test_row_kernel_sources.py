"""Index arithmetic of the row kernels with the launch tables, tile sizes and constants
that their sources state: what `test_row_kernel_index_models` models, read from the code."""
import re
from pathlib import Path

import pytest
import torch

import test_row_kernel_index_models as models
from tempname_5090_b200.ops import actpack, loss, norm

KERNELS = Path(__file__).resolve().parents[1] / "csrc" / "kernels"
JOIN, PACK, SCORE, ROWVEC, API, BIND = ((KERNELS / name).read_text() for name in (
    "join.cu", "actpack.cu", "score.cu", "rowvec.cuh", "kernels_api.h", "kernels_bind.cpp"))
WIDTHS = models.WIDTHS


def value(text, **names):
    """A C++ integer expression of constants, in Python."""
    text = re.sub(r"//.*", "", text)
    text = re.sub(r"\bint64_t\(([^()]*)\)", r"(\1)", text)
    text = re.sub(r"\bint\(([^()]*)\)", r"(\1)", text).replace("::", "_").replace("&&", " and ")
    text = re.sub(r"(?<![/])/(?![/])", "//", text)
    while "?" in text:  # the innermost or last choice first
        m = list(re.finditer(r"([^?:(),]+)\?([^?:(),]+):([^?:(),]+)", text))[-1]
        text = text[:m.start()] + f"(({m[2]}) if ({m[1]}) else ({m[3]}))" + text[m.end():]
    return eval(text, {"__builtins__": {}}, names)


def constant(source, name):
    return value(re.search(rf"\b{name} = ([^,;]+)[,;]", source)[1])


def body(source, head):
    """The text between the braces that follow `head`."""
    at = source.index("{", source.index(head))
    depth = 0
    for i in range(at, len(source)):
        depth += {"{": 1, "}": -1}.get(source[i], 0)
        if not depth:
            return source[at + 1:i]


def table(function, form, size, packed):
    """[(largest width, threads, groups)] of a launch table for values of `size` bytes."""
    text = body(JOIN, function).replace("sizeof(T)", str(size)).replace("!PACKED", str(not packed))
    names = {}
    for name, expression in re.findall(r"constexpr \w+ (\w+) = ([^;]+);", text):
        names[name] = value(expression, **names)
    rows = re.findall(rf"(?:if \(p\.cols <= (\d+)\) )?return {form}<T, ([^;]+)>\(", text)
    limit = constant(API, "kJoinMaxCols")
    out = []
    for most, arguments in rows:
        nt, nv = (value(a, **names) for a in arguments.split(",")[:2])
        out.append((int(most) if most else limit, nt, nv))
    return out


TABLES = {("fwd", size, False): table("int fwd_pick(", "fwd_form", size, False) for size in (2, 4)}
TABLES |= {("bwd", size, packed): table("int bwd_pick(", "bwd_form", size, packed)
           for size in (2, 4) for packed in (False, True)}


def shape(key, cols):
    return next((nt, nv) for most, nt, nv in TABLES[key] if cols <= most)


def test_tables_are_read_as_they_stand():
    for size in (2, 4):
        assert TABLES["fwd", size, False] == models.FWD[size]
        assert TABLES["bwd", size, False] == models.BWD[size]
    # packed FP32 rows have the threads of BF16 rows
    assert TABLES["bwd", 2, True] == TABLES["bwd", 4, True] == models.BWD[2]


@pytest.mark.parametrize("key", list(TABLES), ids=str)
def test_every_width_has_its_columns(key):
    _, size, _ = key
    column = re.search(r"int column\(int g, int i = 0\) \{\s*return FORM \? (.+?) : (.+?);\n", body(JOIN, "struct Tile {"), re.S)
    for cols in range(1, constant(API, "kJoinMaxCols") + 1, 37):
        nt, nv = shape(key, cols)
        assert cols <= nt * nv * 8 and nt % 32 == 0 and nt <= 1024
    for cols in WIDTHS:
        nt, nv = shape(key, cols)
        pieces = size // 2
        names = dict(NT=nt, NV=nv, kPieces=pieces, kPer=8 // pieces,
                     g=torch.arange(nv)[None, :, None], i=torch.arange(8)[None, None, :],
                     tid=torch.arange(nt)[:, None, None])
        for form, vectors in ((column[1], True), (column[2], False)):
            c = value(form.replace("threadIdx.x", "tid"), **names)
            assert torch.equal(c.expand(nt, nv, 8), models.columns(nt, nv, size, vectors))
            assert torch.equal(c.flatten().sort().values, torch.arange(nt * nv * 8))


def sizes(size, nt, nv, form, cols):
    """Bytes of a row's region for values as they are and packed, by the kernels' formulas."""
    pieces = size // 2
    names = dict(NT=nt, NV=nv, kPieces=pieces, cols=cols, FORM=form, sizeof_T=size, row=actpack.row_bytes(cols))

    def of(struct):
        text = re.search(r"int bytes\(int cols\) \{\s*return FORM \? (.+?) : (.+?);\s*\}", body(JOIN, struct), re.S)
        expression = text[1 if form else 2].replace("sizeof(T)", "sizeof_T").replace("pack_row_bytes(cols)", "row")
        return value(expression, **names)

    return of("struct Tile {"), of("struct PackedTile {")


@pytest.mark.parametrize("key", list(TABLES), ids=str)
def test_copies_stay_in_their_regions(key):
    direction, size, packed = key
    pieces, per = size // 2, 16 // size
    for cols in WIDTHS:
        nt, nv = shape(key, cols)
        for form in (0, 1) if cols % 8 == 0 else (0,):
            whole, kept = sizes(size, nt, nv, form, cols)
            if form:
                # a thread's pieces lie k * NT + thread, 16 bytes each
                assert (nv * pieces * nt) * 16 == whole
                # packed: its codes at (k NT + thread) kPer, then the exponents' four bytes
                codes, last = nt * nv * 8, nv * pieces * nt
                assert last * per == codes and codes + last * 4 == kept
                for k in range(nv * pieces):
                    for tid in (0, nt - 1):
                        col = (k * nt + tid) * per
                        if col >= cols:
                            continue
                        first = actpack._align(cols) + (col // 128 & ~3)
                        assert col + per <= actpack._align(cols) and first + 4 <= actpack.row_bytes(cols)
                        assert first % 4 == 0 and col % per == 0 and first <= actpack._align(cols) + col // 128 < first + 4
            else:
                for start in range(0, 16, size):  # the row's first byte in its first piece
                    covered = (start + cols * size + 15) // 16 * 16
                    assert covered <= whole
                assert actpack.row_bytes(cols) <= kept


def test_rings_fit_the_shared_memory():
    most = constant(JOIN, "kMaxRing")
    assert most + 4096 <= 227 * 1024
    stages = {name: constant(JOIN, name) for name in ("kFwdStages", "kBwdStages")}
    for key in TABLES:
        direction, size, packed = key
        for cols in WIDTHS + [5120, 6144, 7168, 8000]:
            nt, nv = shape(key, cols)
            for form in (0, 1) if cols % 8 == 0 else (0,):
                whole, kept = sizes(size, nt, nv, form, cols)
                if direction == "fwd":
                    assert stages["kFwdStages"] * 2 * whole <= most
                else:
                    rows = 1 if size == 4 and nt * nv == 1024 else stages["kBwdStages"]
                    ring = rows * (2 * whole + 2 * (kept if packed else whole))
                    assert ring + nt * nv * (8 * size + 32) <= most


def test_workspace_holds_every_launch():
    text = body(JOIN, "int join_bwd_parts(")
    pick = re.search(r"const int nt = ([^;]+);", text)[1]
    limits = [(int(a), int(b)) for a, b in re.findall(r"cols <= (\d+) \? (\d+)", pick)]
    rest = int(pick.split(":")[-1])
    threads = constant(JOIN, "kSmThreads")
    assert "148 * (kSmThreads / nt)" in text and "std::max(p.rows / (FORM ? 4 : 2), 148)" in JOIN
    for key in TABLES:
        if key[0] == "fwd":
            continue
        for cols in range(1, 8193, 61):
            nt = next((b for a, b in limits if cols <= a), rest)
            used = shape(key, cols)[0]
            for rows in (1, 147, 149, 700, 5000, 10 ** 6):
                for few in (2, 4):
                    assert min(rows, 148 * (threads // used), max(rows // few, 148)) <= min(rows, 148 * (threads // nt))


def test_constants_of_packed_rows_and_the_gelu_table():
    assert constant(ROWVEC, "kPackGroup") == actpack.GROUP
    pad, half, end = (constant(PACK, n) for n in ("kTablePad", "kTableHalf", "kTableEnd"))
    low = constant(PACK, "kTableLow")
    assert (pad, half, end, low - 127) == (48, 256, 64, -24)  # the model's
    assert constant(PACK, "kCopies") == 8 and "(w >> 2) & 0x3fe0u" in PACK and "(w >> 18) & 0x3fe0u" in PACK
    first, count = re.search(r"unit_byte - (\d+)u <= (\d+)u", PACK).groups()
    assert (int(first), int(first) + int(count)) == (112, 126)  # the units that the model goes over
    codes = re.search(r"pack_code_bytes\(int64_t cols\) \{ return ([^;]+);", ROWVEC)[1]
    for cols in WIDTHS + [129, 50304]:
        assert value(codes, cols=cols) == actpack._align(cols)


def test_parts_of_a_clusters_row():
    step, most = "((vocab + C - 1) / C + step - 1) / step * step", re.search(r"while \(C < (\d+) &&", SCORE)[1]
    assert step in SCORE and most == "4"
    for vocab in (8192, 8193, 20001, 32003, 50304):
        for C in (2, 4):
            for per in (4, 8):
                chunk = value(step, vocab=vocab, C=C, step=per)
                assert chunk % per == 0 and (C - 1) * chunk < vocab <= C * chunk


def test_limits_of_python_and_kernels_agree():
    assert constant(API, "kJoinMaxCols") == norm.JOIN_MAX_COLS
    assert constant(SCORE, "kMaxTop") == loss.MAX_TOP
    assert f"top_k <= {loss.MAX_TOP} && top_k <= vocab" in BIND


def test_limits_of_the_fast_sums():
    """The rounding of R = fl(m log2 e) that the sums carry stays below 1 for every running
    maximum, and what is counted at the start or lifted to the floor vanishes in a row that
    counts: 2^t is zero below t = -126."""
    floor, low, plain = (float(re.search(rf"{n} = ([0-9.]+)f", SCORE)[1]) for n in ("kFloor", "kLow", "kPlain"))
    assert (floor, low, plain) == (2.0 ** 25, 2.0 ** 24, 2.0 ** 22)
    log2e = float(torch.tensor(1.44269504088896340736))
    m = torch.cat([torch.linspace(-low, plain, 200001), torch.tensor([-low, -plain, plain])]).float()
    exact = m.double() * log2e
    off = exact - exact.float().double()
    assert off.abs().max() <= 1 and off[m >= -plain].abs().max() <= 0.25
    assert (-floor + low) * log2e + 1 < -126 and (-low + plain) * log2e + 1 < -126
    bf16_floor = int(re.search(r"floor\(\) \{ return 0x([0-9a-f]{4})\1u; \}  // -kFloor", SCORE)[1], 16)
    bits = torch.tensor([bf16_floor - 0x10000], dtype=torch.int16)
    assert bits.view(torch.bfloat16).item() == -floor


def test_native_entries_have_callers():
    """No entry of the row operators that neither the package nor a test calls."""
    names = re.findall(r'm\.def\("(\w+)"', BIND)
    names = names[names.index("ce_bwd") + 1:names.index("grad_sqsum_parts")]
    root = KERNELS.parents[1]
    text = "".join(p.read_text() for folder in ("tempname_5090_b200", "tests") for p in (root / folder).rglob("*.py"))
    assert "token_logprobs" in names and [n for n in names if f"lib().{n}(" not in text] == []
