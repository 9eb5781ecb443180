"""Host side and source of the operators around the GEMMs, without a GPU."""
import re
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "355_1_trans_b200" / "csrc"


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
