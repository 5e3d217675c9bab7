"""CPU tests of the reading operators: the boundary of libartread.so and every refusal, none of which may
reach a GPU."""
import ctypes
import os
import re
import struct
import subprocess

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from art_amd import reader as rd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _declared():
    with open(os.path.join(ROOT, "include", "artread.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    return sorted(set(re.findall(r"\b(artread_[a-z_]+)\s*\(", text)))


def test_header_binding_and_library_agree():
    assert _declared() == sorted(rd.READ_SYMBOLS)
    lib = ctypes.CDLL(rd.READ_LIB_PATH)
    for name in _declared():
        assert getattr(lib, name) is not None
    # seven pointers, eighteen int64, int32 + float; one pointer, three int64, three pointers
    assert ctypes.sizeof(rd.AttendArgs) == 25 * 8 + 8
    assert ctypes.sizeof(rd.AttendGrads) == 7 * 8
    a, g = _attend(), rd.AttendGrads(*range(1, 8))
    assert rd._pack_args(*(getattr(a, n) or 0 for n, _ in a._fields_)) == bytes(a)
    assert rd._pack_grads(*range(1, 8)) == bytes(g)


# ---- the Python layer -----------------------------------------------------------------------------
TOKENS = torch.zeros((3, 5), dtype=torch.int32)
TABLE = torch.zeros((7, 8), dtype=torch.float16)
LENS = torch.full((3,), 5, dtype=torch.int32)


@pytest.mark.parametrize("kwargs", [
    dict(tokens=TOKENS.float()),
    dict(tokens=TOKENS.short()),
    dict(lengths=LENS.long()),
    dict(lengths=LENS[:2]),
    dict(lengths=LENS[:, None]),
    dict(table=TABLE.double()),
    dict(table=TABLE.int()),
    dict(table=TABLE[0]),
    dict(table=TABLE.t()),
    dict(table=TABLE[:1].expand(7, 8)),
    dict(table=TABLE[:0]),
    dict(out_dtype=torch.float32),
    dict(out_dtype=torch.bfloat16),
    dict(table=TABLE.float(), out_dtype=torch.float64),
    dict(scale=float("nan")),
    dict(scale=float("inf")),
    dict(scale=1e39),
    dict(vocab_base=1 << 63),
    dict(),  # all fine, but not on a GPU
], ids=str)
def test_embed_tokens_refuses(kwargs):
    args = dict(tokens=TOKENS, table=TABLE, lengths=LENS)
    args.update(kwargs)
    with pytest.raises(ValueError):
        rd.embed_tokens(**args)


@pytest.mark.parametrize("kwargs", [
    dict(grad_out=torch.zeros((3, 5, 8), dtype=torch.float64)),
    dict(grad_out=torch.zeros((3, 4, 8), dtype=torch.float16)),
    dict(grad_out=torch.zeros((3, 5), dtype=torch.float16)),
    dict(vocab=0),
    dict(vocab=1 << 31),
    dict(dtype=torch.bfloat16),
    dict(lengths=LENS.long()),
    dict(scale=float("inf")),
    dict(),
], ids=str)
def test_embed_tokens_grad_refuses(kwargs):
    args = dict(grad_out=torch.zeros((3, 5, 8), dtype=torch.float16), tokens=TOKENS, vocab=7, lengths=LENS)
    args.update(kwargs)
    with pytest.raises(ValueError):
        rd.embed_tokens_grad(**args)


def test_rows_of_more_than_the_limit_are_refused_by_name():
    wide = torch.zeros((1, rd.MAX_ROW + 8), dtype=torch.float16)
    tokens = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="at most"):
        rd.embed_tokens(tokens, wide)
    with pytest.raises(ValueError, match="at most"):
        rd.embed_tokens_grad(wide[None], tokens, 1)


Q = torch.zeros((2, 3, 4, 16), dtype=torch.float16)
K = torch.zeros((2, 5, 6, 2, 16), dtype=torch.float16)
KL = torch.zeros((2, 5), dtype=torch.int32)


@pytest.mark.parametrize("kwargs", [
    dict(query=Q[0]),
    dict(key=K[0, 0], value=K[0, 0]),
    dict(value=K[:, :4]),
    dict(query=Q.float()),
    dict(query=Q.float(), key=K.float(), value=K.float()),
    dict(value=K.bfloat16()),
    dict(query=Q[:1]),
    dict(query=Q[..., :8]),
    dict(query=Q[..., :12], key=K[..., :12], value=K[..., :12]),
    dict(query=torch.zeros((2, 3, 4, 136), dtype=torch.float16), key=torch.zeros((2, 5, 6, 2, 136), dtype=torch.float16),
         value=torch.zeros((2, 5, 6, 2, 136), dtype=torch.float16)),
    dict(query=Q[:, :, :3]),
    dict(key=K[:, :, :, :0], value=K[:, :, :, :0]),
    dict(lengths=KL.long()),
    dict(lengths=KL[0]),
    dict(lengths=KL[:, :4]),
    dict(scale=float("nan")),
    dict(scale=float("-inf")),
    dict(),
], ids=lambda k: ",".join(sorted(k)))
def test_cross_attention_refuses(kwargs):
    args = dict(query=Q, key=K, value=K, lengths=KL)
    args.update(kwargs)
    with pytest.raises(ValueError):
        rd.cross_attention(**args)


LSE = torch.zeros((2, 4, 3))


@pytest.mark.parametrize("kwargs", [
    dict(grad_out=Q[:, :2]),
    dict(grad_out=Q.bfloat16()),
    dict(out=Q.transpose(1, 2).contiguous().transpose(1, 2)),
    dict(out=Q[:1]),
    dict(saved=(LSE.half(), Q)),
    dict(saved=(LSE.transpose(1, 2), Q)),
    dict(saved=(torch.zeros((2, 3, 4)).transpose(1, 2), Q)),
    dict(saved=(LSE, Q.bfloat16())),
    dict(saved=(LSE, Q[:1])),
    dict(lengths=KL.long()),
    dict(),
], ids=lambda k: ",".join(sorted(k)))
def test_cross_attention_grad_refuses(kwargs):
    args = dict(grad_out=Q, query=Q, key=K, value=K, out=Q, saved=(LSE, Q), lengths=KL)
    args.update(kwargs)
    with pytest.raises(ValueError):
        rd.cross_attention_grad(**args)


@pytest.mark.parametrize("which", ["table", "query", "key", "value", "grad_out", "embed grad_out", "out", "rest"])
def test_forward_mode_tangents_are_refused(which):
    """A call by address sees a dual tensor's values only: its tangent would be gone from the result."""
    forward_ad = torch.autograd.forward_ad

    def call(dual):
        if which == "table":
            return rd.embed_tokens(TOKENS, dual(TABLE), LENS)
        if which == "embed grad_out":
            return rd.embed_tokens_grad(dual(torch.zeros((3, 5, 8), dtype=torch.float16)), TOKENS, 7, LENS)
        args = dict(query=Q, key=K, value=K, lengths=KL)
        if which in args:
            args[which] = dual(args[which])
            return rd.cross_attention(**args)
        return rd.cross_attention_grad(dual(Q) if which == "grad_out" else Q, out=dual(Q) if which == "out" else Q,
                                       saved=(LSE, dual(Q) if which == "rest" else Q), **args)

    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError):   # without a tangent: on past it, to the tensors' place
            call(lambda t: t)


CALLS = {
    "embed_tokens": (lambda t, w: rd.embed_tokens(t, w), (TOKENS, TABLE)),
    "embed_tokens_grad": (lambda g, t: rd.embed_tokens_grad(g, t, 7), (torch.zeros((3, 5, 8)), TOKENS)),
    "cross_attention": (lambda q, k: rd.cross_attention(q, k, k), (Q, K)),
    "cross_attention_grad": (lambda q, k: rd.cross_attention_grad(q, q, k, k, q, (LSE, q)), (Q, K)),
}


@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    """A recorded graph would hold the allocation of the outputs and no call: its replay would return what is in memory."""
    call, args = CALLS[name]
    with pytest.raises(NotImplementedError):
        torch.jit.trace(call, args, check_trace=False)
    with pytest.raises(NotImplementedError):
        make_fx(call)(*args)
    with pytest.raises(ValueError):   # not traced: on past it, to the tensors' place
        call(*args)


# ---- the C entry points: refused before the device is even looked at -------------------------------
SOME = 4096  # an address that is never followed


def _embed_args(**change):
    a = dict(device=0, table=SOME, table_dtype=0, vocab=7, dim=8, stride=8, tokens=SOME, token_bytes=4, lengths=None,
             n=3, len=5, base=0, scale=1.0, out=SOME, out_dtype=0, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [
    dict(table=None), dict(out=None), dict(tokens=None), dict(token_bytes=2), dict(n=0), dict(len=0), dict(n=-1),
    dict(n=1 << 20, len=1 << 11), dict(n=1 << 40, len=1 << 40), dict(vocab=0), dict(vocab=1 << 31), dict(dim=0),
    dict(dim=(1 << 20) + 1), dict(stride=7), dict(table_dtype=3), dict(out_dtype=2), dict(out_dtype=-1),
    dict(table_dtype=1, out_dtype=0), dict(table=SOME + 1), dict(tokens=SOME + 2), dict(lengths=SOME + 2), dict(scale=float("nan")),
], ids=str)
def test_c_embed_refuses(change):
    assert rd._read().artread_embed(*_embed_args(**change)) == -1
    assert rd._read().artread_last_error()


@pytest.mark.parametrize("change", [
    dict(grad=None), dict(table=None), dict(ws=None), dict(ws=SOME + 4), dict(bytes=0), dict(bytes=-1), dict(n=0),
    dict(vocab=0), dict(dim=0), dict(table_dtype=1), dict(grad_dtype=5), dict(token_bytes=1), dict(scale=float("inf")),
], ids=str)
def test_c_embed_grad_refuses(change):
    need = rd._read().artread_embed_grad_workspace(7, 8, 3, 5)
    assert need > 0
    a = dict(device=0, grad=SOME, grad_dtype=0, tokens=SOME, token_bytes=4, lengths=None, n=3, len=5, vocab=7, dim=8,
             base=0, scale=1.0, table=SOME, table_dtype=0, ws=SOME, bytes=need, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    assert rd._read().artread_embed_grad(*a.values()) == -1


def test_c_workspace_sizes():
    lib = rd._read()
    for bad in ((0, 8, 3, 5), (7, 0, 3, 5), (7, 8, 0, 5), (7, 8, 3, 0), (7, 8, 1 << 20, 1 << 11), (1 << 31, 8, 3, 5)):
        assert lib.artread_embed_grad_workspace(*bad) == -1
    # two lists of (key, position), partial sums of at most two rows of 8 to 64 positions each, vocabulary marks
    n, dim, vocab = 2048 * 256, 768, 30522
    size = lib.artread_embed_grad_workspace(vocab, dim, 2048, 256)
    assert 2 * 8 * n <= size <= 2 * 8 * n + (n // 8 + 1) * 2 * dim * 4 + 5 * vocab + (1 << 20)


def _attend(**change):
    a = dict(q=SOME, k=SOME, v=SOME, lengths=None, out=SOME, lse=SOME, rest=None, batch=2, rows=3, passages=5, len=6, heads=4,
             kv_heads=2, dim=16, q_batch=192, q_row=64, q_head=16, k_batch=960, k_passage=192, k_row=32, k_head=16,
             v_batch=960, v_passage=192, v_row=32, v_head=16, dtype=0, scale=0.25)
    assert set(change) <= set(a)
    a.update(change)
    return rd.AttendArgs(*a.values())


BAD_ATTEND = [
    dict(dtype=2), dict(batch=0), dict(rows=0), dict(passages=0), dict(len=0), dict(heads=0), dict(kv_heads=0),
    dict(kv_heads=3), dict(dim=0), dict(dim=12), dict(dim=136), dict(rows=1 << 31), dict(batch=1 << 20, rows=1 << 20),
    dict(passages=1 << 20, len=1 << 20), dict(batch=1, passages=1, len=(1 << 31) - 1, kv_heads=1, heads=1), dict(scale=float("nan")), dict(q_row=-8), dict(k_row=12),
    dict(v_batch=1 << 40), dict(k_row=1 << 24), dict(v_row=1 << 24), dict(q_row=1 << 24), dict(q_head=1 << 28),
]


@pytest.mark.parametrize("change", BAD_ATTEND + [dict(q=None), dict(k=None), dict(v=None), dict(out=None),
                                                 dict(q=SOME + 8), dict(lse=SOME + 2), dict(lengths=SOME + 1), dict(out=SOME + 2), dict(rest=SOME + 8)], ids=str)
def test_c_attend_refuses(change):
    lib, a = rd._read(), _attend(**change)
    if change in BAD_ATTEND:
        assert lib.artread_attend_workspace(ctypes.byref(a)) == -1
        assert lib.artread_attend_grad_workspace(ctypes.byref(a)) == -1
    assert lib.artread_attend(0, ctypes.byref(a), SOME, 1 << 40, None) == -1
    g = rd.AttendGrads(SOME, 192, 64, 16, SOME, SOME, SOME)
    assert lib.artread_attend_grad(0, ctypes.byref(a), ctypes.byref(g), SOME, 1 << 40, None) == -1


def test_c_attend_grad_refuses():
    lib, a = rd._read(), _attend()
    need = lib.artread_attend_grad_workspace(ctypes.byref(a))
    assert need > 0
    fine = dict(grad_out=SOME, g_batch=192, g_row=64, g_head=16, grad_q=SOME, grad_k=SOME, grad_v=SOME)
    for change in (dict(grad_out=None), dict(grad_q=None), dict(grad_k=None), dict(grad_v=None), dict(g_row=-8),
                   dict(g_row=4), dict(g_row=1 << 24), dict(g_head=1 << 28), dict(grad_v=SOME + 8)):
        g = rd.AttendGrads(*dict(fine, **change).values())
        assert lib.artread_attend_grad(0, ctypes.byref(a), ctypes.byref(g), SOME, need, None) == -1, change
    g = rd.AttendGrads(*fine.values())
    for ws, size in ((None, need), (SOME, need - 1), (SOME + 8, need)):
        assert lib.artread_attend_grad(0, ctypes.byref(a), ctypes.byref(g), ws, size, None) == -1
    no_lse = _attend(lse=None)
    assert lib.artread_attend_grad(0, ctypes.byref(no_lse), ctypes.byref(g), SOME, need, None) == -1
    assert lib.artread_attend(0, None, None, 0, None) == -1
    assert lib.artread_attend_workspace(None) == -1


# ---- what was compiled ------------------------------------------------------------------------------
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _gpu_code(tmp_path):
    """{kernel: instructions} of the built library's gfx950 code."""
    with open(rd.READ_LIB_PATH, "rb") as f:
        data = f.read()
    at = data.index(b"__CLANG_OFFLOAD_BUNDLE__")
    (count,), place = struct.unpack_from("<Q", data, at + 24), at + 32
    for _ in range(count):
        offset, size, chars = struct.unpack_from("<QQQ", data, place)
        target = data[place + 24:place + 24 + chars]
        place += 24 + chars
        if target.endswith(b"gfx950"):
            code = tmp_path / "artread.co"
            code.write_bytes(data[at + offset:at + offset + size])
    text = subprocess.run([OBJDUMP, "-d", str(code)], check=True, capture_output=True, text=True).stdout
    kernels, name = {}, None
    for line in text.splitlines():
        head = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if head:
            name = head.group(1)
            kernels[name] = []
        elif name and line.startswith("\t"):
            kernels[name].append(line.split("//")[0].strip())
    return kernels


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_cleared_tiles_are_settled_before_memory_is_loaded_into_them(tmp_path):
    """The few-row gradient clears the wave's own tiles by LDS stores and then loads memory into them: loads to LDS do
    not wait for LDS stores by themselves, so a wait for all of these stands between the two."""
    seen = 0
    for name, code in _gpu_code(tmp_path).items():
        if "attend_grad_stream_kernel" not in name:
            continue
        seen += 1
        load = next(i for i, x in enumerate(code) if x.startswith("global_load_lds"))
        store = max(i for i, x in enumerate(code[:load]) if x.startswith("ds_write"))
        assert any(re.match(r"s_waitcnt lgkmcnt\(0\)$", x) for x in code[store:load]), name
    assert seen == 12
