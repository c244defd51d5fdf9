"""The register report reads every kernel that ptxas names."""
from results_b200.utils import ptxas_report

TEXT = """ptxas info    : 0 bytes gmem
ptxas info    : Compiling entry function '_Z1kPf' for 'sm_100a'
ptxas info    : Function properties for _Z1kPf
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used 10 registers, used 1 barriers
ptxas info    : Compile time = 3.944 ms
ptxas info    : Compiling entry function '_Z1mPf' for 'sm_100a'
ptxas info    : Function properties for _Z1mPf
    8 bytes stack frame, 12 bytes spill stores, 16 bytes spill loads
ptxas info    : Used 64 registers, used 1 barriers, 8 bytes cumulative stack size, 464 bytes smem
ptxas info    : Function properties for _Z4waitv
    24 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
"""


def test_kernels_with_and_without_static_shared_memory():
    a, b = ptxas_report.parse(TEXT)
    assert (a["name"], a["regs"], a["smem"], a["spill_st"]) == ("k(float*)", 10, 0, 0)
    assert (b["name"], b["regs"], b["smem"], b["stack"], b["spill_st"], b["spill_ld"]) == ("m(float*)", 64, 464, 8, 12, 16)
