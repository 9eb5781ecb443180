"""Host side and source of the operators around the GEMMs, without a GPU."""
import ctypes
import importlib
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "355_1_trans_b200" / "csrc"


@pytest.fixture(scope="module")
def host_arith(tmp_path_factory):
    """host_arith.cu, the library's host arithmetic, as a shared library of its own."""
    nvcc = importlib.import_module("355_1_trans_b200.build").nvcc()
    lib = tmp_path_factory.mktemp("host_arith") / "libhost_arith.so"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "--expt-relaxed-constexpr",
                    "-Xcompiler", "-fPIC,-fvisibility=hidden", "-shared", "-cudart", "static", "-ccbin",
                    shutil.which("g++") or "g++", "-I", str(ROOT / "include"), "-o", str(lib),
                    str(ROOT / "tests" / "host_arith.cu")], check=True, capture_output=True, text=True)
    return lib


@pytest.mark.parametrize("fp4", [0, 1])
@pytest.mark.parametrize("kernel", ["auto", "1cta", "swap", "pair"])
def test_plan_of_a_short_contraction(bs, host_arith, fp4, kernel):
    """A K of less than one stage is planned without a division by its zero stages (in a
    child: the division would end the process), and longer ones have no empty slice."""
    code = """if True:
        import ctypes, sys
        lib, out = ctypes.CDLL(sys.argv[1]), (ctypes.c_longlong * 3)()
        for m in (1, 64, 300):
            for k in (32, 64, 96, 128, 192, 256, 512, 7168):
                for split in (0, 1, 4, 64):
                    lib.plan_mx(m, 256, k, int(sys.argv[2]), int(sys.argv[3]), split, 148, out)
                    kb, s, per = out
                    assert kb == k // (256 if int(sys.argv[2]) else 128), (m, k, split, list(out))
                    assert s >= 1 and per >= 1 and s * per >= kb, (m, k, split, list(out))
                    assert (s - 1) * per < max(kb, 1), (m, k, split, list(out))
    """
    r = subprocess.run([sys.executable, "-c", code, str(host_arith), str(fp4), str(bs.KERNELS[kernel])],
                       capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)


def test_written_data_is_not_read_as_read_only():
    """What an operator reads, a kernel that may still run when it starts has written, or
    it writes itself (in place): nothing of it is loaded through the read-only path."""
    norm = (CSRC / "layer_norm.cuh").read_text()
    quant = (CSRC / "quant.cuh").read_text()
    for text in (norm, (CSRC / "epilogue.cuh").read_text(), quant[quant.index("struct DequantParams"):]):
        code = re.sub(r"//.*", "", text)
        assert not re.search(r"__ldg\s*\(|\.nc\b", code)


def test_copies_beside_a_kernel_read_past_l1():
    """A dequantise that has not waited for the writers of its operands loads at GPU scope."""
    text = (CSRC / "quant.cuh").read_text()
    loads = re.findall(r"template <bool kBeside>\n__device__ __forceinline__ \w+ (\w+)\(const uint8_t\* p\) \{(.*?)\n\}", text,
                       re.S)
    assert len(loads) == 3
    assert all("if constexpr (!kBeside)" in body and "ld.relaxed.gpu.global" in body for _, body in loads)
    piece = text[text.index("void dequantize_piece("):text.index("__global__ void __launch_bounds__(256) dequantize_kernel")]
    reads = re.findall(r"(?:raw\[k\]|raw\[k\]\.x|scale\[k\]) = (?!make_uint2|0u)(\w+)<kBeside>", piece)
    assert sorted(reads) == sorted(name for name, _ in loads)


@pytest.mark.parametrize("stages", [2, 3, 5, 8])
def test_ring_copies_in_flight(host_arith, stages):
    """When a wait of the layer norm gradient's ring runs out, exactly the copies that were
    issued and not yet waited for are waited for, at the parity that each completes."""
    lib = ctypes.CDLL(str(host_arith))
    out = (ctypes.c_int * 32)()
    for step in (1, 7, 148):
        for count in (1, 2, stages - 1, stages, stages + 1, 3 * stages + 1):
            rows, row0 = (count - 1) * step + 1 + step // 2, step // 2   # this CTA's rows: `count` of them
            issued = {}                                                 # stage -> turns whose copies it was given
            for turn in range(min(stages, count)):
                issued.setdefault(turn % stages, []).append(turn)
            stage = phase = 0
            for turn in range(count):   # the wait of this turn runs out
                # the n-th copy into a stage completes its barrier's n-th phase, of parity n % 2
                want = {s: (len(turns) - 1) % 2 for s, turns in issued.items() if turns[-1] >= turn}
                n = lib.ring_pending(row0 + turn * step, step, rows, stages, stage, phase, out)
                assert n == len(want) and {out[2 * i]: out[2 * i + 1] for i in range(n)} == want, (step, count, turn)
                # or it does not: the stage takes the row `stages` turns on
                if turn + stages < count:
                    issued[stage].append(turn + stages)
                stage += 1
                if stage == stages:
                    stage, phase = 0, phase ^ 1
    with_source = (CSRC / "layer_norm.cuh").read_text()
    assert "ring.drain(row, step, p.rows, p.timeout_ns)" in with_source
