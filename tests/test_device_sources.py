"""CPU test of the GPU code's text: instruction families that no device source of the tree may hold, in any form (inline
assembly, builtins, assembly files) and wherever it lies -- a stand-alone probe that nothing builds counts like the library.

Data is written through vector stores only.  The scalar data cache is not coherent with them, so a write through it (a scalar
store, a scalar atomic, a write-back or discard of that cache) can lose or overtake the vector stores beside it.

Single-precision arithmetic is written one value per lane: some forms of the packed instructions (two f32 per instruction) have
given wrong results on MI355X now and then, without an error.  The compiler makes them from ordinary float code too, so the
built libraries' device code is looked at as well."""
import os
import re
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = re.compile(r"\.(hip|cu|cpp|cc|c|hpp|h|cuh|s|S|ll|py|sh|txt|cmake|mk)$|^Makefile$")
FOLDERS = ("timemachine_amd", "include", "oracle", "scripts", "tests", "bench.py", "__graft_entry__.py")
SCALAR_CACHE_WRITE = re.compile(r"(?:\b|_)s_(?:(?:scratch_|buffer_)?(?:store|atomic)_|dcache_(?:wb|discard))", re.IGNORECASE)
PACKED_F32 = re.compile(r"\bv_pk_(?:add|mul|fma)_f32\b", re.IGNORECASE)


def device_sources():
    for top in FOLDERS:
        path = os.path.join(REPO, top)
        if os.path.isfile(path):
            yield path
        for folder, _, files in os.walk(path):
            for f in files:
                if SOURCE.search(f):
                    yield os.path.join(folder, f)


def hits(pattern, path):
    with open(path, errors="replace") as fh:
        return [f"{os.path.relpath(path, REPO)}:{n}: {line.strip()}" for n, line in enumerate(fh, 1) if pattern.search(line)]


@pytest.mark.parametrize("op", ["store_dword", "atomic_add", "buffer_store_dwordx2", "scratch_store_dword", "buffer_atomic_or", "dcache_wb", "dcache_discard_x2"])
def test_the_scalar_cache_pattern_finds_every_kind_of_write(op):
    assert SCALAR_CACHE_WRITE.search(f'asm volatile("s_{op} %0, %1, 0x0")')
    assert SCALAR_CACHE_WRITE.search(f"__builtin_amdgcn_s_{op}();")


@pytest.mark.parametrize("op", ["s_load_dword", "s_buffer_load_dwordx4", "s_waitcnt lgkmcnt(0)", "ds_add_u64", "global_store_dword", "global_atomic_add_x2", "buffer_store_dword", "is_store_", "s_dcache_inv"])
def test_the_scalar_cache_pattern_leaves_loads_and_vector_stores(op):
    assert not SCALAR_CACHE_WRITE.search(f'asm volatile("{op} %0, %1")')


def test_no_source_writes_through_the_scalar_data_cache():
    found = [h for path in device_sources() for h in hits(SCALAR_CACHE_WRITE, path)]
    assert not found, "\n".join(found)


@pytest.mark.parametrize("op", ["add", "mul", "fma"])
def test_the_packed_f32_pattern_finds_every_kind(op):
    assert PACKED_F32.search(f'asm volatile("v_pk_{op}_f32 %0, %0, %1" : "+v"(a))')
    assert not PACKED_F32.search(f'asm volatile("v_pk_{op}_f16 %0, %0, %1" : "+v"(a))')
    assert not PACKED_F32.search(f'asm volatile("v_{op}_f32 %0, %0, %1" : "+v"(a))')


def test_no_source_holds_packed_f32_arithmetic():
    found = [h for path in device_sources() for h in hits(PACKED_F32, path)]
    assert not found, "\n".join(found)


@pytest.mark.parametrize("lib", ["libtimemachine_amd.so", "libtimemachine_amd_rowblock.so"])
def test_the_built_device_code_holds_no_packed_f32_arithmetic(lib, tmp_path):
    objdump = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
    src = os.path.join(REPO, "timemachine_amd", "csrc", lib)
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(src):
        import __graft_entry__

        __graft_entry__.build()
    copy = shutil.copy(src, tmp_path)
    subprocess.run([objdump, "--offloading", copy], check=True, stdout=subprocess.DEVNULL)  # writes the code objects beside the copy
    objects = sorted(p for p in tmp_path.iterdir() if "amdgcn" in p.name)
    assert len(objects) >= 5
    total = 0
    for obj in objects:
        text = subprocess.run([objdump, "-d", str(obj)], check=True, capture_output=True, text=True).stdout
        total += text.count("v_fma_f32") + text.count("v_mul_f32")
        packed = PACKED_F32.findall(text)
        assert not packed, f"{obj.name}: {len(packed)} packed f32 instructions"
    assert total > 1000  # the listing is one of the f32 kernels too


LOAD = re.compile(r"\b(?:ds_read|ds_load|global_load|flat_load|buffer_load|scratch_load|s_load|s_buffer_load)\w*")
COMMENT = re.compile(r"//[^\n]*|/\*.*?\*/", re.DOTALL)


def asm_statements(text):
    """the argument lists of the inline asm statements, comments taken out"""
    text = COMMENT.sub("", text)
    for m in re.finditer(r"\b(?:asm|__asm__)\b\s*(?:volatile|__volatile__)?\s*\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        yield text[m.end():i - 1]


def loads_without_their_wait(text):
    # a statement may name its instructions through macros, and those through others
    macros = dict(re.findall(r"#define (\w+)(?:\([^)]*\))?((?:[^\n]*\\\n)*[^\n]*)", COMMENT.sub("", text)))
    loading = {m for m, body in macros.items() if LOAD.search(body)}
    while True:
        more = {m for m, body in macros.items() if any(re.search(rf"\b{k}\b", body) for k in loading)} | loading
        if more == loading:
            break
        loading = more
    return [s for s in asm_statements(text) if (LOAD.search(s) or any(re.search(rf"\b{k}\b", s) for k in loading)) and "s_waitcnt" not in s]


def test_the_search_for_loads_without_their_wait():
    read = 'ds_read_b64 %0, %1 offset:8'
    assert loads_without_their_wait(f'asm volatile("{read}" : "=v"(v) : "v"(a)); asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v));')
    assert not loads_without_their_wait(f'asm volatile("{read}\\n\\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(a));')
    assert not loads_without_their_wait(f'// asm volatile("{read}")\nasm volatile("v_mov_b32 %0, %1" : "=v"(v) : "v"(a)); // {read}')
    macro = f'#define READ(C) "{read}\\n\\t"\n#define READ_ALL READ(0) \\\n    READ(1)\n'
    assert loads_without_their_wait(macro + 'asm volatile(READ_ALL : "=v"(v) : "v"(a));')
    assert not loads_without_their_wait(macro + 'asm volatile(READ_ALL "s_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(a));')


def test_every_load_in_inline_asm_is_waited_for_in_its_own_statement():
    """The compiler takes an asm output as written when the statement ends: a load still under way behind it lands in a register
    that may have been copied or given away meanwhile."""
    found = []
    for path in device_sources():
        if path.endswith((".hip", ".hpp", ".h", ".cpp")):
            with open(path, errors="replace") as fh:
                found += [f"{os.path.relpath(path, REPO)}: {s}" for s in loads_without_their_wait(fh.read())]
    assert not found, "\n".join(found)
