"""What the compiler made of the kernels, read in the assembly it prints for them, and the host side of what
the kernels compute with (no GPU needed)."""
import concurrent.futures
import os
import re
import subprocess

import pytest

from fused_attention_amd import build

HIPCC = os.path.join(build.ROCM, "bin", "hipcc")

# (head_dim, blocks of 16 rows per wave, key groups): two and three ring slots, one and two key groups, one sub-tile at a time
# and two.  The registers that a kernel may have come from where the launcher takes them.
GROUP_KERNELS = [(16, 1, 1), (16, 1, 2), (32, 1, 1), (32, 1, 2), (32, 2, 1), (64, 1, 1), (128, 1, 1), (128, 1, 2)]
ELEMENTS = ["fp16", "bf16"]


@pytest.fixture(scope="module")
def group_kernels(tmp_path_factory):
    """{(element, head_dim, NQ, GK, mode): ([lines of the kernel's assembly], {what its metadata say})}, unmasked (mode 0) and
    causal (2)."""
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    where = tmp_path_factory.mktemp("asm")

    def compiled(element):
        space = "fa::bf16" if element == "bf16" else "fa"
        source = ['#include "%s"' % os.path.join(build.CSRC, "fused_attn_kernel.hpp")]
        source += ["template __global__ void %s::fwd_kernel_group<%d, %d, %d, fa::%s, fa::group_waves_per_simd<%d, %d, false>()>(const fa::SplitParams);"
                   % (space, h, nq, gk, mode, h, nq) for h, nq, gk in GROUP_KERNELS for mode in ("kPlain", "kCausal")]
        (where / (element + ".hip")).write_text("\n".join(source) + "\n")
        subprocess.run([HIPCC] + build.HIPCC_FLAGS + ["--cuda-device-only", "-S", str(where / (element + ".hip")), "-o", str(where / (element + ".s"))],
                       check=True, capture_output=True)
        return (where / (element + ".s")).read_text()

    with concurrent.futures.ThreadPoolExecutor() as pool:
        texts = dict(zip(ELEMENTS, pool.map(compiled, ELEMENTS)))
    kernels = {}
    name = r"_ZN2fa(?:4bf16)?16fwd_kernel_groupILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)E"
    for element, text in texts.items():
        lines = None
        for line in text.splitlines():
            found = re.match(name + r"\w+:", line)
            if found:
                lines = []
                kernels[(element,) + tuple(int(n) for n in found.groups())] = lines, {}
            elif line.startswith(".Lfunc_end"):
                lines = None
            elif lines is not None:
                lines.append(line.strip())
        for entry in text[text.index("amdhsa.kernels:"):].split("  - .agpr_count:")[1:]:
            found = re.search(r"\.name: +" + name, entry)
            kernels[(element,) + tuple(int(n) for n in found.groups())][1].update(
                (key, int(n)) for key, n in re.findall(r"\.(private_segment_fixed_size|vgpr_spill_count|vgpr_count): +(\d+)", entry))
    return kernels


def _loop_lines(lines):
    """The instructions of the blocks that the compiler marks as part of a loop, without those written by hand."""
    in_loop = by_hand = False
    for line in lines:
        if re.match(r"(\.LBB\d+_\d+:|; %bb\.)", line):
            in_loop = False
        in_loop = in_loop or (line.startswith((";", ".LBB")) and "Loop" in line)
        by_hand = "#ASMSTART" in line or (by_hand and "#ASMEND" not in line)
        if in_loop and not by_hand and line[:1] not in (";", ".", ""):
            yield line


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("H,NQ,GK", GROUP_KERNELS)
@pytest.mark.parametrize("element", ELEMENTS)
def test_the_group_kernel_waits_for_its_queries_once(group_kernels, H, NQ, GK, mode, element):
    # The key tiles come by loads written in assembly, with exact waits of their own, so that the only loads the compiler
    # knows of are the queries'.  A wait of its making inside a loop would be one for the key tiles on their way, in every pass.
    lines, _ = group_kernels[element, H, NQ, GK, mode]
    assert any("s_barrier" in line for line in _loop_lines(lines))
    assert [line for line in _loop_lines(lines) if line.startswith("s_waitcnt") and "vmcnt" in line] == []


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("H,NQ,GK", GROUP_KERNELS)
@pytest.mark.parametrize("element", ELEMENTS)
def test_the_group_kernel_keeps_its_values_in_registers(group_kernels, H, NQ, GK, mode, element):
    # None of its values pass through memory, with as many waves per SIMD as the launcher compiles it for (64 registers with
    # eight, 80 with six, 128 with four).
    _, said = group_kernels[element, H, NQ, GK, mode]
    assert said["private_segment_fixed_size"] == said["vgpr_spill_count"] == 0
    assert said["vgpr_count"] <= (64 if NQ == 1 and H <= 32 else 80 if NQ == 1 and H <= 64 else 128)


def test_division_by_multiplication_is_exact(tmp_path):
    # fa::Divisor as the kernels use it (the high half of n * mul, shifted), at every d up to 70, at every power of
    # two and its neighbours, and at the largest one: n on both sides of multiples of d, over the whole range.
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    (tmp_path / "div.hip").write_text('#include "%s"\n' % os.path.join(build.CSRC, "fused_attn_kernel.hpp") + r"""
#include <cstdio>
int main() {
    const int64_t most = 0x7fffffff;
    auto check = [&](int64_t d) {
        const fa::Divisor by = fa::divisor(d);
        auto right = [&](int64_t n) {
            const int64_t got = by.mul == 0 ? n : (int64_t)((((uint64_t)n * by.mul) >> 32) >> by.shift);
            if (got != n / d) std::printf("%lld / %lld is not %lld\n", (long long)n, (long long)d, (long long)got);
            return got == n / d;
        };
        const int64_t whole = most / d, step = whole / 1000 + 1;
        for (int64_t i = 0; i <= whole; i += step)
            for (int64_t n = i * d - 1; n <= i * d + 1; ++n)
                if (n >= 0 && n <= most && !right(n)) return false;
        for (int64_t n = whole * d - 1; n <= most && n <= whole * d + 1; ++n)
            if (n >= 0 && !right(n)) return false;
        return right(0) && right(d - 1) && right(most - 1) && right(most);
    };
    for (int64_t d = 1; d <= 70; ++d)
        if (!check(d)) return 1;
    for (int s = 1; s <= 31; ++s)
        for (int64_t d = ((int64_t)1 << s) - 1; d <= ((int64_t)1 << s) + 1 && d <= most; ++d)
            if (!check(d)) return 1;
    return check(most) ? 0 : 1;
}
""")
    subprocess.run([HIPCC] + build.HIPCC_FLAGS + [str(tmp_path / "div.hip"), "-o", str(tmp_path / "div")], check=True, capture_output=True)
    ran = subprocess.run([str(tmp_path / "div")], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout


# (kernel, template arguments): keys through LDS in each width and form of the rows; histograms of one wave
CACHE_KERNELS = [("cached_attention_kernel", "%d, %s, %d, %d, fa::cache::%s" % at) for at in (
    (32, "false", 1, 4, "kEvery"), (64, "true", 2, 4, "kEvery"), (128, "false", 1, 8, "kListed"), (128, "true", 1, 1, "kListed"),
    (64, "false", 1, 2, "kShared"))] + [("select_pages_rows_kernel", "64, false")]


def test_lanes_that_exchange_through_lds_do_so_in_order(tmp_path):
    # Where the lanes of a wave read what others of it wrote, no instruction is needed between, but the compiler must not exchange the
    # two either: between stores, counts and loads there is a barrier, of the workgroup or of the wave.
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    params = {"cached_attention_kernel": "AttendParams", "select_pages_rows_kernel": "SelectParams"}
    source = ['#include "%s"' % os.path.join(build.CSRC, "cache_kernels.hpp")]
    source += ["template __global__ void fa::cache::%s<%s>(const fa::cache::%s);" % (name, at, params[name]) for name, at in CACHE_KERNELS]
    (tmp_path / "cache.hip").write_text("\n".join(source) + "\n")
    subprocess.run([HIPCC] + build.HIPCC_FLAGS + ["--cuda-device-only", "-S", str(tmp_path / "cache.hip"), "-o", str(tmp_path / "cache.s")],
                   check=True, capture_output=True)
    checked = 0
    kernel = last = None
    by_wave = False
    for line in (tmp_path / "cache.s").read_text().splitlines():
        found = re.match(r"_ZN2fa5cache\d+(cached_attention_kernel|select_pages_rows_kernel)\w+:", line)
        if found:
            kernel, last, by_wave = line, None, False
        elif line.startswith(".Lfunc_end"):
            checked += kernel is not None and by_wave
            kernel = None
        elif kernel is not None:
            text = line.strip()
            if "s_barrier" in text or "wave barrier" in text:
                last = None
                by_wave = by_wave or "wave barrier" in text
            # the exchanged ones: keys and the histogram's words, 8 or 16 bytes at a time, and its counts
            op = re.match(r"ds_(read_b64|read_b128|write_b64|write_b128|add_u32)", text)
            if op:
                kind = op.group(1).split("_")[0]
                assert last in (None, kind), (kernel, text)
                last = kind
    assert checked == len(CACHE_KERNELS)


def test_no_exception_leaves_a_c_entry(tmp_path):
    # The host side alone, with a HIP runtime that does nothing and no memory to be had: launches that opt into more LDS and would
    # remember that they did return a status all the same, every time.
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    (tmp_path / "main.cpp").write_text(r"""
#include <cstdio>
#include <cstdlib>
#include <new>
#include "fused_attn.h"
static bool memory = true;
static int opted = 0, launched = 0;
void* operator new(std::size_t n) {
    void* p = memory ? std::malloc(n) : nullptr;
    if (p == nullptr) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }
extern "C" {
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void*, int, int) { ++opted; return 0; }
struct Dim { unsigned x, y, z; };
int hipLaunchKernel(const void*, Dim, Dim, void**, std::size_t, void*) { ++launched; return 0; }
void** __hipRegisterFatBinary(const void*) { static void* handle; return &handle; }
void __hipRegisterFunction(...) {}
void __hipUnregisterFatBinary(void**) {}
int __hipPopCallConfiguration(...) { return 0; }
int hipEventCreate(...) { return 0; }
int hipEventDestroy(...) { return 0; }
int hipEventRecord(...) { return 0; }
int hipEventSynchronize(...) { return 0; }
int hipEventElapsedTime(...) { return 0; }
const char* hipGetErrorString(int) { return ""; }
}
int main() {
    alignas(16) static char room[64];
    const int32_t* n = reinterpret_cast<const int32_t*>(room);
    fa_cache c = {room, room, room, room, room, n, 1000, 8, 64, 128, 1, 100, 100};
    for (int i = 0; i < 6; ++i) {
        memory = i >= 3;
        const int before = opted;
        const int many = fa_cached_attention(&c, room, 0, 128, 4096, room, 0, 128, 4096, nullptr, nullptr, 0, n, nullptr, 2000, 32, 1.f, 1,
                                             room, (int64_t)1 << 40, nullptr);
        const int listed = fa_cached_attention(&c, room, 0, 128, 4096, room, 0, 128, 4096, nullptr, n, 40, n, nullptr, 2, 32, 1.f, 1,
                                               room, (int64_t)1 << 40, nullptr);
        const int select = fa_select_pages(&c, room, 0, 128, 4096, reinterpret_cast<int32_t*>(room), 4, n, nullptr, 1, 32, 0, nullptr);
        const int dense = fa_fwd(room, room, room, nullptr, room, 8, 32, 4096, 128, 32 * 4096 * 128, 4096 * 128, 128, 0.1f, nullptr);
        std::printf("%d %d %d %d, %d\n", many, listed, select, dense, opted - before);
    }
    std::printf("%d\n", launched);
}
""")
    objects = []
    for name in build.LIB_SOURCES:
        objects.append(str(tmp_path / (name + ".o")))
        subprocess.run([HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O1", "-w", "-fPIC", "--cuda-host-only", "-c", os.path.join(build.CSRC, name), "-o",
                        objects[-1]], check=True, capture_output=True)
    subprocess.run(["g++", "-std=c++17", "-w", "-I" + os.path.join(build.REPO_DIR, "include"), str(tmp_path / "main.cpp")] + objects +
                   ["-Wl,--unresolved-symbols=ignore-in-object-files", "-o", str(tmp_path / "main")], check=True, capture_output=True)
    ran = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stderr
    lines = ran.stdout.split("\n")
    statuses, asked = zip(*(line.split(", ") for line in lines[:6]))
    assert set(statuses) == {"0 0 0 0"}, lines
    # asked for until there is memory to remember it, and then no more
    assert min(int(n) for n in asked[:4]) >= 4 and asked[4:] == ("0", "0"), lines
    assert int(lines[6]) >= 24


def test_the_cache_kernels_keep_their_values_in_registers(tmp_path):
    # None of their values pass through scratch memory but for those of the lists at head_dim 128 with one and four waves, which are
    # compiled for three waves a SIMD: at most 16 bytes a lane.
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    attend = [(h, nq, waves, rows) for h in (64, 128) for nq, waves, rows in (
        (1, 4, "kEvery"), (2, 4, "kEvery"), (1, 8, "kListed"), (1, 4, "kListed"), (1, 1, "kListed"), (1, 4, "kShared"), (1, 2, "kShared"))]

    def compiled(element):
        source = ['#include "%s"' % os.path.join(build.CSRC, "cache_kernels.hpp")]
        source += ["template __global__ void fa::cache::cached_attention_kernel<%d, %s, %d, %d, fa::cache::%s>(const fa::cache::AttendParams);" %
                   (h, element, nq, waves, rows) for h, nq, waves, rows in attend]
        source += ["template __global__ void fa::cache::cached_attention_wide_kernel<%d, %s, %d>(const fa::cache::AttendParams);" % (h, element, nq)
                   for h in (64, 128) for nq in (1, 2)]
        (tmp_path / (element + ".hip")).write_text("\n".join(source) + "\n")
        subprocess.run([HIPCC] + build.HIPCC_FLAGS + ["--cuda-device-only", "-S", str(tmp_path / (element + ".hip")), "-o", str(tmp_path / (element + ".s"))],
                       check=True, capture_output=True)
        text = (tmp_path / (element + ".s")).read_text()
        return text[text.index("amdhsa.kernels:"):].split("  - .agpr_count:")[1:]

    with concurrent.futures.ThreadPoolExecutor() as pool:
        entries = sum(pool.map(compiled, ("false", "true")), [])
    assert len(entries) == 2 * (len(attend) + 4)
    for entry in entries:
        name = re.search(r"\.name: +(\S+)", entry).group(1)
        scratch = int(re.search(r"\.private_segment_fixed_size: +(\d+)", entry).group(1))
        # (kListed is 1)
        may = re.search(r"cached_attention_kernelILi128ELb[01]ELi1ELi[14]ELNS0_4RowsE1E", name) is not None
        assert scratch <= (16 if may else 0), (name, scratch)
