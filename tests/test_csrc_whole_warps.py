"""Instructions that a warp has to run as a whole (.aligned), as far as the kernels' sources show: lanes that have left a loop one after the other meet before them."""
import pathlib
import re

CSRC = pathlib.Path(__file__).parents[1] / "isca-2025-lia_b200" / "csrc"
SOURCES = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu*"))}


def test_clusters_meet_by_whole_warps():
    """A cluster's barrier stands in two functions, and in both the warp meets right before it: callers come from loops over threadIdx.x."""
    found = [(name, m.start()) for name, text in SOURCES.items() for m in re.finditer(r"barrier\.cluster\.arrive", text)]
    assert [name for name, _ in found] == ["common.cuh", "umma.cuh"]
    for name, at in found:
        body = SOURCES[name][SOURCES[name].rindex("{", 0, at):at]
        assert re.match(r'\{\s*__syncwarp\(\);\s*asm volatile\("$', body), (name, body)


def test_tmem_of_products_in_8_bits_is_given_back_by_whole_warps():
    """The parts of a tile are added up in loops whose rounds differ from lane to lane; the warp that gives TMEM back has left them together."""
    text = SOURCES["int8_gemm_sm100.cu"]
    loop = text.rindex("i < last * 4; i += 256")
    assert "__syncwarp();" in text[loop:text.index("tcgen05.dealloc", loop)].split("if (*dead)")[0]
