"""The vocabulary operators without a GPU: the C ABI's symbols and struct, host arithmetic, argument
refusals at the three levels (C ABI, direct handles, operators)."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
ONE = 0x1000  # an aligned address that no refused call reads


def test_header_symbols_all_exported_and_bound(native_libs):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "rafhip_vocab.h").read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(rafhip_[a-z0-9_]+)\s*\(", text)))
    lib = native_libs.optim()
    for n in names:
        assert hasattr(lib, n), f"{n} declared in rafhip_vocab.h but not exported"
    assert sorted(native_libs.VOCAB_SYMBOLS) == names
    assert int(re.search(r"#define\s+RAFHIP_MAX_TOPK\s+(\d+)", text).group(1)) == native_libs.RAFHIP_MAX_TOPK


def test_argument_struct_layout_matches_the_header(native_libs, tmp_path):
    import subprocess

    fields = [f[0] for f in native_libs.TopkDistillArgs._fields_]
    src = tmp_path / "layout.c"
    prints = "".join(f'printf("%zu ", offsetof(rafhip_topk_distill_args, {f}));' for f in fields)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "rafhip_vocab.h"\nint main(void) {' + prints +
                   'printf("%zu", sizeof(rafhip_topk_distill_args)); return 0; }')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(native_libs.TopkDistillArgs, f).offset for f in fields] + [ctypes.sizeof(native_libs.TopkDistillArgs)]
    assert got == want


def test_embedding_dx_workspace(native_libs):
    ws = native_libs.optim().rafhip_embedding_dx_workspace_bytes
    assert ws(0, 100, 8) == ws(1, 100, 8) == ws(5000, 0, 8) == ws(5000, 8, 0) == 0
    last = 0
    for n in (1000, 5000, 70_000, 300_000, 8_388_608):
        assert ws(n, 50257, 64) >= max(last, 4 * n)
        last = ws(n, 50257, 64)
    # the partial sums are a sixteenth of the tokens at most, rows and runs a few words per token
    assert last < 8_388_608 * (4 * 64 / 16 + 24)
    assert ws(8_388_609, 50257, 64) == -1 and ws(8_388_608, 262_143, 64) > 0 and ws(8_388_608, 262_144, 64) == -1
    assert ws(1 << 20, (1 << 21) - 1, 1) > 0 and ws((1 << 20) + 1, (1 << 21) - 1, 1) == -1
    assert ws(1, 1 << 21, 1) == -1 and b"1 tokens over 2097152 rows of width 1" in native_libs.optim().rafhip_last_error()
    assert ws(1, 1, 1) == 0 and native_libs.optim().rafhip_last_error() == b""  # nor is an older message left
    assert ws(-1, 1, 1) == -1 and ws(1, -1, 1) == -1 and ws(1, 1, 1 << 24) == -1


def test_embedding_argument_validation(native_libs):
    L = native_libs
    f, dx = L.optim().rafhip_embedding, L.optim().rafhip_embedding_dx
    good = [ONE, L.RAFHIP_F32, 10, 4, ONE, 64, 3, 0, 1.0, ONE, L.RAFHIP_F32, None]

    def call(fn, args, **change):
        a = list(args)
        for at, v in change.items():
            a[int(at[1:])] = v
        return fn(*a)

    assert call(f, good, _6=0) == 0 and call(f, good, _3=0) == 0  # nothing to do
    for change in ({"_6": -1}, {"_2": -1}, {"_3": -1}, {"_7": -1}, {"_0": None}, {"_4": None}, {"_9": None}, {"_0": ONE + 2},
                   {"_9": ONE + 1}, {"_4": ONE + 4}, {"_7": (1 << 63) - 5}):
        assert call(f, good, **change) == L.RAFHIP_ERR_INVALID_ARG, change
    for change in ({"_1": L.RAFHIP_F64}, {"_10": 7}, {"_5": 16}, {"_3": 1 << 24}):
        assert call(f, good, **change) == L.RAFHIP_ERR_UNSUPPORTED, change
    #        0    1           2    3   4     5   6  7  8  9  10   11   12         13 14   15 16
    good = [ONE, L.RAFHIP_BF16, ONE, 32, 5000, 10, 4, 0, 0, 0, 1.0, ONE, L.RAFHIP_F32, 0, ONE, 1 << 30, None]
    assert call(dx, good, _5=0) == 0 and call(dx, good, _6=0) == 0
    assert call(dx, good, _4=0, _13=1) == 0  # no token adds nothing
    for change in ({"_4": -1}, {"_0": None}, {"_2": None}, {"_11": None}, {"_0": ONE + 1}, {"_2": ONE + 2}, {"_11": ONE + 2},
                   {"_7": -3}):
        assert call(dx, good, **change) == L.RAFHIP_ERR_INVALID_ARG, change
    for change in ({"_1": 3}, {"_12": 9}, {"_3": 8}, {"_5": 1 << 21}, {"_4": 1 << 24}):
        assert call(dx, good, **change) == L.RAFHIP_ERR_UNSUPPORTED, change
    for change in ({"_14": None}, {"_15": 100}, {"_14": ONE + 8}):
        assert call(dx, good, **change) == L.RAFHIP_ERR_WORKSPACE, change
        assert b"workspace" in L.optim().rafhip_last_error()


def _args(L, **change):
    a = dict(logits=ONE, topk_indices=ONE, topk_logits=ONE, labels=ONE, rows=4, vocab=50257, row_stride=50304, topk=8,
             logits_dtype=L.RAFHIP_BF16, topk_dtype=L.RAFHIP_F32, index_bits=64, temperature=2.0, soft_weight=1.0,
             hard_weight=0.5)
    a.update(change)
    return L.TopkDistillArgs(**a)


def test_distill_argument_validation(native_libs):
    L = native_libs
    lib = L.optim()
    ws = lambda a: lib.rafhip_topk_distill_workspace_bytes(ctypes.byref(a))
    assert ws(_args(L)) > 0 and ws(_args(L, rows=4096)) == 0 and ws(_args(L, rows=0)) == 0
    assert ws(_args(L, rows=4096, vocab=210_000, row_stride=210_000)) == 4096 * 16 * 7  # longer than the registers hold
    assert lib.rafhip_topk_distill_workspace_bytes(None) == -1

    def all_three(a, loss=ONE, stats=ONE, dloss=ONE, count=4, out=ONE, width=50304, space=ONE, nbytes=1 << 20):
        p = ctypes.byref(a)
        return (lib.rafhip_topk_distill(p, loss, stats, space, nbytes, None),
                lib.rafhip_topk_distill_dx(p, dloss, count, stats, out, width, None),
                lib.rafhip_topk_distill_step(p, dloss, count, loss, out, width, space, nbytes, None))

    bad, no, space = L.RAFHIP_ERR_INVALID_ARG, L.RAFHIP_ERR_UNSUPPORTED, L.RAFHIP_ERR_WORKSPACE
    for change in (dict(rows=-1), dict(vocab=-1), dict(topk=-1), dict(row_stride=50256), dict(temperature=0.0),
                   dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                   dict(temperature=1e-40), dict(temperature=3.5e-39), dict(soft_weight=float("nan")), dict(hard_weight=float("inf")),
                   dict(logits=None), dict(topk_indices=None), dict(topk_logits=None), dict(logits=ONE + 1),
                   dict(topk_indices=ONE + 4), dict(topk_logits=ONE + 2), dict(labels=ONE + 4)):
        assert all_three(_args(L, **change)) == (bad, bad, bad), change
        assert ws(_args(L, **change)) == -1 or "logits" in change or "topk_indices" in change or "topk_logits" in change \
            or "labels" in change
    for change in (dict(logits_dtype=L.RAFHIP_F64), dict(topk_dtype=9), dict(index_bits=16), dict(topk=1025),
                   dict(vocab=1 << 28, row_stride=1 << 28), dict(row_stride=1 << 28)):
        assert all_three(_args(L, **change)) == (no, no, no), change
    assert all_three(_args(L, rows=0), count=0) == (0, 0, 0)
    p = ctypes.byref(_args(L, vocab=70_000, row_stride=70_000))  # four rows, read in parts
    assert lib.rafhip_topk_distill(p, None, ONE, ONE, 1 << 20, None) == bad
    assert lib.rafhip_topk_distill(p, ONE, ONE, None, 0, None) == space
    assert lib.rafhip_topk_distill(p, ONE, ONE, ONE, 64, None) == space
    assert lib.rafhip_topk_distill(p, ONE, ONE, ONE + 8, 1 << 20, None) == space
    for kw in (dict(count=3), dict(count=0), dict(dloss=None), dict(out=None), dict(width=50256), dict(out=ONE + 1),
               dict(dloss=ONE + 2)):
        assert all_three(_args(L), loss=None, **kw)[1:] == (bad, bad), kw
    assert lib.rafhip_topk_distill_dx(p, ONE, 4, None, ONE, 70_016, None) == bad
    assert lib.rafhip_topk_distill_step(p, ONE, 4, ONE, ONE, 70_016, None, 0, None) == space
    for fn in (lib.rafhip_topk_distill, lib.rafhip_topk_distill_dx, lib.rafhip_topk_distill_step):
        assert fn(None, *[None if t is ctypes.c_void_p else 0 for t in fn.argtypes[1:]]) == bad


def test_outputs_that_share_bytes_are_refused(native_libs):
    """Each output against each input and the other outputs: its first byte on the other's last, its last
    on the other's first, and both in one place."""
    L = native_libs
    lib, f32, bf16 = L.optim(), L.RAFHIP_F32, L.RAFHIP_BF16
    ws = 1 << 24

    def refused(call, sizes, outs):
        far = {name: (i + 1) << 32 for i, name in enumerate(sizes)}
        for o in outs:
            for other in sizes:
                if other == o or not sizes[o] or not sizes[other]:
                    continue
                for at in (far[other] + sizes[other] - 16, far[other] - sizes[o] + 16, far[other]):
                    at -= at % 16  # the workspace's alignment, and everything's
                    if not (at < far[other] + sizes[other] and far[other] < at + sizes[o]):
                        at = far[other]
                    assert call(**{**far, o: at}) == L.RAFHIP_ERR_INVALID_ARG, (o, other)
                    message = lib.rafhip_last_error().decode()
                    assert f"{o} overlaps {other}" in message or f"{other} overlaps {o}" in message, message

    refused(lambda x, indices, y: lib.rafhip_embedding(x, f32, 100, 64, indices, 64, 50, 0, 1.0, y, bf16, None),
            {"x": 100 * 64 * 4, "indices": 400, "y": 50 * 64 * 2}, ["y"])
    need = lib.rafhip_embedding_dx_workspace_bytes(5000, 100, 64)
    refused(lambda dy, indices, dx, workspace: lib.rafhip_embedding_dx(dy, bf16, indices, 32, 5000, 100, 64, 0, 0, 0, 1.0, dx, f32,
                                                                        1, workspace, need, None),
            {"dy": 5000 * 64 * 2, "indices": 20000, "dx": 100 * 64 * 4, "workspace": need}, ["dx", "workspace"])
    refused(lambda dy, indices, dx: lib.rafhip_embedding_dx(dy, bf16, indices, 32, 200, 100, 64, 0, 0, 0, 1.0, dx, f32, 0, None, 0,
                                                            None),
            {"dy": 200 * 64 * 2, "indices": 800, "dx": 100 * 64 * 4}, ["dx"])

    def args(logits, topk_indices, topk_logits, labels):
        return ctypes.byref(_args(L, rows=40, vocab=70_000, row_stride=70_016, topk=8, logits=logits, topk_indices=topk_indices,
                                  topk_logits=topk_logits, labels=labels))

    ins = {"logits": (39 * 70_016 + 70_000) * 2, "topk_indices": 40 * 64, "topk_logits": 40 * 32, "labels": 320}
    need = lib.rafhip_topk_distill_workspace_bytes(ctypes.byref(_args(L, rows=40, vocab=70_000, row_stride=70_016)))
    assert 0 < need < ws
    refused(lambda loss, stats, workspace, **t: lib.rafhip_topk_distill(args(**t), loss, stats, workspace, ws, None),
            {**ins, "loss": 160, "stats": 480, "workspace": need}, ["loss", "stats", "workspace"])
    refused(lambda dloss, stats, dlogits, **t: lib.rafhip_topk_distill_dx(args(**t), dloss, 40, stats, dlogits, 70_001, None),
            {**ins, "dloss": 160, "stats": 480, "dlogits": 40 * 70_001 * 2}, ["dlogits"])
    refused(lambda dloss, loss, dlogits, workspace, **t: lib.rafhip_topk_distill_step(args(**t), dloss, 40, loss, dlogits, 70_001,
                                                                                      workspace, ws, None),
            {**ins, "dloss": 160, "loss": 160, "dlogits": 40 * 70_001 * 2, "workspace": need}, ["loss", "dlogits", "workspace"])


def test_declares_reach_python(native_libs):
    from raf_amd import _lib, op

    for name in ("embedding", "embedding_dx", "topk_distill", "topk_distill_dx", "topk_distill_step"):
        assert op.dispatch_list(f"raf.op.{name}") == [("hip", f"raf.op.hip.{name}", 30)]
    x, ids = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    z, top, t = torch.zeros(4, 9), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    stats = torch.zeros(4, 3)
    refused = [
        ("no valid dispatch|Cannot find a valid dispatch for op raf.op.embedding:", lambda: op.embedding(x, ids)),
        ("a table of rows", lambda: op.embedding(x[0], ids)),
        ("int32 or int64", lambda: op.embedding(x, ids.to(torch.int16))),
        ("first_row", lambda: op.embedding(x, ids, first_row=-1)),
        ("Cannot find a valid dispatch for op raf.op.embedding_dx", lambda: op.embedding_dx(torch.zeros(3, 8), ids, 5)),
        ("one dimension more", lambda: op.embedding_dx(torch.zeros(3, 1, 8), ids, 5)),
        ("differ in shape", lambda: op.embedding_dx(torch.zeros(4, 8), ids, 5)),
        ("num_weight must not", lambda: op.embedding_dx(torch.zeros(3, 8), ids, -5)),
        ("num_weight rows", lambda: op.embedding_dx(torch.zeros(3, 8), ids, 5, grad=torch.zeros(4, 8))),
        ("output's dtype", lambda: op.embedding_dx(torch.zeros(3, 8), ids, 5, out_dtype=torch.float16, grad=torch.zeros(5, 8))),
        ("Cannot find a valid dispatch for op raf.op.topk_distill:", lambda: op.topk_distill(z, top, t)),
        ("the logits' rows", lambda: op.topk_distill(z, top[:3], t[:3])),
        ("differ in shape", lambda: op.topk_distill(z, top, t[:, :1].contiguous())),
        ("int32 or int64", lambda: op.topk_distill(z, t, t)),
        ("vocab_size", lambda: op.topk_distill(z, top, t, vocab_size=10)),
        ("labels must have the logits' rows", lambda: op.topk_distill(z, top, t, labels=top)),
        ("dtype of topk_indices", lambda: op.topk_distill(z, top, t, labels=torch.zeros(4, dtype=torch.int64))),
        ("dloss must have", lambda: op.topk_distill_step(z, top, t, torch.zeros(3))),
        ("dloss must be float32", lambda: op.topk_distill_step(z, top, t, torch.zeros(4, dtype=torch.float16))),
        ("stats must be", lambda: op.topk_distill_dx(torch.zeros(4), z, top, t, torch.zeros(4, 2))),
        ("Cannot find a valid dispatch for op raf.op.topk_distill_dx", lambda: op.topk_distill_dx(torch.zeros(1), z, top, t, stats)),
    ]
    for message, call in refused:
        with pytest.raises(_lib.RafError, match=message):
            call()
    with pytest.raises(ValueError, match="contiguous"):
        op.embedding(x.t(), ids)
    with pytest.raises(TypeError, match="expected a tensor"):
        op.embedding(x, [1, 2])
    with pytest.raises(TypeError, match="out_dtype"):
        op.embedding(x, ids, out_dtype=torch.complex64)


def test_integers_beyond_64_bits_are_refused_not_cut(native_libs):
    from raf_amd import op

    x, ids = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    z, top, t = torch.zeros(4, 9), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    dy, wraps = torch.zeros(3, 8), 1 << 64
    for name, call in (("first_row", lambda: op.embedding(x, ids, first_row=wraps)),
                       ("first_row", lambda: op.embedding_dx(dy, ids, 5, first_row=wraps + 1)),
                       ("num_weight", lambda: op.embedding_dx(dy, ids, wraps + 5)),
                       ("padding_idx", lambda: op.embedding_dx(dy, ids, 5, padding_idx=1 - wraps)),
                       ("vocab_size", lambda: op.topk_distill(z, top, t, vocab_size=wraps + 9)),
                       ("vocab_size", lambda: op.topk_distill_step(z, top, t, torch.zeros(4), vocab_size=wraps))):
        with pytest.raises(ValueError, match=f"{name}: .* does not fit 64 bits"):
            call()


def test_direct_handles_refuse_cpu_tensors():
    from raf_amd import kernels

    x, ids = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        kernels.embedding(x, ids)
    with pytest.raises(ValueError, match="GPU"):
        kernels.embedding_dx(torch.zeros(3, 8), ids, x)
    with pytest.raises(ValueError, match="GPU"):
        kernels.TopkDistill(x, ids.reshape(1, 3), x[:1, :3])


def test_keys_tell_calls_apart(native_libs):
    key = native_libs.glue().key
    a, b = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    keys = [key(t) for t in ((a,), (b,), (a, None), (None, a), (a, a), (a.reshape(3, 2),), (a.reshape(6),), (a.half(),),
                             (a.bfloat16(),), (torch.zeros(2, 3, 1),), (torch.zeros(()),), ())]
    assert len(set(keys)) == len(keys)
    assert key((a, b)) == key((torch.ones(2, 3), torch.ones(2, 3, dtype=torch.int32)))
    for bad, error in (([a], TypeError), ((a,) * 9, TypeError), ((1,), TypeError), ((a.t(),), ValueError),
                       ((torch.zeros(2, dtype=torch.complex64),), TypeError)):
        with pytest.raises(error):
            key(bad)
