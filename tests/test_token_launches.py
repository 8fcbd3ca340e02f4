"""The launches of the token operators, without a GPU: a small program whose own
functions stand in for HIP's records them.  A launch has fewer than 2^32
threads along each axis, and one that is refused is not followed by those that
read its results."""
import subprocess

import pytest

import hip_oracles
from conftest import ROOT


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    program = tmp_path_factory.mktemp("recorder") / "launch_recorder"
    subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic",
                    str(ROOT / "tests" / "launch_recorder.cpp"), str(hip_oracles.LIB_PATH),
                    f"-Wl,-rpath,{hip_oracles.LIB_PATH.parent}", "-Wl,--allow-shlib-undefined",
                    "-o", str(program)], check=True, capture_output=True)

    def run(op, *numbers, fail=-1):
        """([(kernel, grid, block)], return code)"""
        out = subprocess.run([str(program), str(fail), op, *map(str, numbers)], check=True,
                             capture_output=True, text=True).stdout.splitlines()
        made = [line.split() for line in out[:-1]]
        return ([(m[0], tuple(map(int, m[1:4])), tuple(map(int, m[4:7]))) for m in made],
                int(out[-1].split()[1]))

    return run


def assert_launchable(made):
    for kernel, grid, block in made:
        assert block[0] * block[1] * block[2] <= 1024, (kernel, block)
        assert grid[1] <= 65535 and grid[2] <= 65535 and min(grid) > 0, (kernel, grid)
        assert all(g * b < 1 << 32 for g, b in zip(grid, block)), (kernel, grid, block)


@pytest.mark.parametrize("out", [2, 4])
@pytest.mark.parametrize("vocab", [(1 << 30), (1 << 29) + 1, 1 << 29, 10 ** 7, 32000])
@pytest.mark.parametrize("count,width", [(1, 17), (1, 32), (1025, 8), (2000, 4096), (0, 1 << 20),
                                         (70001, 1 << 16)])
def test_embedding_gradients_of_large_vocabularies(count, width, vocab, out, launches):
    for accumulate in (0, 1):
        made, rc = launches("embedding_bwd", count, width, vocab, 2, out, accumulate)
        assert rc == 0 and (made or count == 0)
        assert_launchable(made)


@pytest.mark.parametrize("accumulate", [0, 1])
def test_a_refused_launch_ends_an_embedding_gradient(accumulate, launches):
    """sum_rows reads the order that the sort writes, and the pieces that are
    joined are sum_rows's."""
    call = ("embedding_bwd", 2000, 64, 5000, 2, 4, accumulate)
    made, rc = launches(*call)
    assert rc == 0 and len(made) == len({kernel for kernel, _, _ in made}) == 3
    for n in range(3):
        again, rc = launches(*call, fail=n)
        assert rc == 9 and again == made[:n + 1]


def test_a_refused_launch_ends_sliced_log_probabilities(launches):
    call = ("token_logprobs", 2, 1 << 20, 2, 8)
    made, rc = launches(*call)
    assert rc == 0 and len(made) == 2
    again, rc = launches(*call, fail=0)
    assert rc == 9 and again == made[:1]


def test_the_widest_embedding_gradients(launches):
    """Columns are counted in 32 bits, up to a workgroup's columns past the last."""
    most = (1 << 31) - 4097
    for elem in (2, 4):
        pieces = -(-most * elem // 16)
        made, rc = launches("embedding_bwd", 33, most, 3, elem, 4, 1)
        assert rc == 0
        assert_launchable(made)
        # 33 places, and the sums of two pieces of 32 in two forms.
        lanes = sum(grid[0] * block[0] for kernel, grid, block in made if "sum_rows" in kernel)
        assert lanes >= pieces * (33 + 2 * 2)
        for width in (most + 1, (1 << 31) - 1):
            made, rc = launches("embedding_bwd", 33, width, 3, elem, 4, 1)
            assert rc == 1000 and not made


def test_a_rows_threads_change_at_whole_rounds_of_loads(launches):
    """Rows few enough for 1024 threads get them where 256 threads with four
    16-byte loads each take more than three rounds."""
    for elem in (2, 4):
        per_round = 256 * 4 * 16 // elem
        for rows in (1, 100, 256):
            for rounds in (2, 3, 4, 5):
                threads = 256 if rounds < 4 else 1024
                for vocab in ((rounds - 1) * per_round + 16 // elem, rounds * per_round):
                    made, rc = launches("token_logprobs", rows, vocab, elem, 0)
                    assert rc == 0 and [m[1:] for m in made] == [((rows, 1, 1), (threads, 1, 1))]
