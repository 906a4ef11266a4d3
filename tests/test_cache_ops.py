"""The operators around an evicting cache without a GPU: their descriptors' layouts, and that
every call they do not take is refused before anything is launched."""
import ctypes
import os
import re
import subprocess

import llm_hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {
    "llh_qk_rope_desc": llm_hip.QkRopeDesc,
    "llh_kv_select_desc": llm_hip.KvSelectDesc,
    "llh_kv_compact_desc": llm_hip.KvCompactDesc,
}


def test_descriptor_layouts_match_header(tmp_path):
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "llm_hip.h"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        src.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        for field, _ in py._fields_:
            src.append(f'  printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));')
    src.append("  return 0; }")
    c, exe = tmp_path / "probe.c", tmp_path / "probe"
    c.write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    got = dict()
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, val = line.split()
        got[cname, field] = int(val)
    for cname, py in STRUCTS.items():
        assert got[cname, "size"] == ctypes.sizeof(py), cname
        for field, _ in py._fields_:
            assert got[cname, field] == getattr(py, field).offset, (cname, field)


def test_constants_match_header():
    text = open(os.path.join(ROOT, "include", "llm_hip.h")).read()
    assert int(re.search(r"#define LLH_WEIGHTS_MAX_CHUNK (\d+)", text).group(1)) == llm_hip.WEIGHTS_MAX_CHUNK
    for name, val in re.findall(r"LLH_(ROPE_[A-Z]+) = (\d+)", text):
        assert getattr(llm_hip, name) == int(val)


def test_refused_calls(tmp_path):
    """tests/cache_refusals.cpp: host objects in the place of a context and a pool."""
    exe = tmp_path / "refusals"
    libs = os.path.dirname(llm_hip.LIB_PATH)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(
        ["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I",
         os.path.join(ROOT, "kir-ai_amd", "csrc"), "-isystem", os.path.join(rocm, "include"),
         os.path.join(ROOT, "tests", "cache_refusals.cpp"), "-o", str(exe), llm_hip.LIB_PATH, "-L",
         os.path.join(rocm, "lib"), "-lamdhip64", "-lpthread", f"-Wl,-rpath,{libs}:{rocm}/lib"], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr


def test_workspace_bound():
    """A decode step's scores alone are 4 bytes a (head, token)."""
    lib = llm_hip.load_library()
    assert lib.llh_weights_workspace_bytes(4, 1, 16, 128, 1000) >= 4 * 16 * 1000 * 4
    assert lib.llh_weights_workspace_bytes(4, 8, 16, 128, 1000) >= 8 * 4 * 16 * 1000 * 4
    assert lib.llh_weights_workspace_bytes(4, 0, 16, 128, 1000) == 0


def test_binding_refuses_rows_it_would_misread():
    """Tensors of another shape, type or order than the library walks, before any call reaches it."""
    import types

    import pytest
    import torch

    ctx = llm_hip.Context.__new__(llm_hip.Context)
    ctx.handle = None  # nothing below gets as far as the library
    i32 = dict(dtype=torch.int32)
    pool = types.SimpleNamespace(info=types.SimpleNamespace(kv_heads=4), handle=None)
    lens, w = torch.zeros(2, **i32), torch.zeros(2, 4, 64)
    desc = types.SimpleNamespace(num_seqs=2)
    ctx._check_weights(pool, desc, None, w)
    ctx._check_weights(pool, desc, w, w)
    for w_in, w_out in [(None, w[:1]), (None, w[:, :2].contiguous()), (None, w.reshape(8, 64)), (w[..., :32], w),
                        (None, w.double()), (None, w.transpose(0, 1)), (w[:1], w)]:
        with pytest.raises(llm_hip.LlhError):
            ctx._check_weights(pool, desc, w_in, w_out)

    keep, kept = torch.zeros(2, 4, 16, **i32), torch.zeros(2, **i32)
    select = ctx.select_desc(lens, 4, 64, 16, 0, 0, 64, 16)
    for bad in [dict(weights=w[:1]), dict(weights=w.half()), dict(weights=w[..., ::2]), dict(keep=keep[:, :3].contiguous()),
                dict(keep=keep.long()), dict(keep=keep.transpose(0, 1)), dict(kept_lens=kept[:1]),
                dict(kept_lens=kept.long())]:
        with pytest.raises(llm_hip.LlhError):
            ctx.kv_select(select, **dict(dict(weights=w, keep=keep, kept_lens=kept), **bad))

    good = dict(seq_lens=lens, kept_lens=kept, keep=keep, src_tables=torch.zeros(2, 4, **i32),
                dst_tables=torch.zeros(2, 1, **i32), max_kept=16, weights_in=w, weights_out=w.clone())
    move = ctx.compact_desc(**good)
    for bad in [dict(keep=keep[0]), dict(keep=keep[:1]), dict(keep=keep.long()), dict(kept_lens=kept[:1]),
                dict(src_tables=good["src_tables"].long()), dict(src_tables=good["src_tables"][:, ::2]),
                dict(dst_tables=good["dst_tables"][:1]), dict(weights_in=w.double()),
                dict(weights_out=torch.zeros(2, 2, 64)), dict(weights_in=w[0])]:
        with pytest.raises(llm_hip.LlhError):
            ctx.compact_desc(**dict(good, **bad))
    pool.info.kv_heads = 2
    with pytest.raises(llm_hip.LlhError):
        ctx.kv_compact(pool, move)
