"""Which kernel the tests of the linear with adapters run, on the host: a change of the rule between the two must not leave one of them
without the tests that were written for it."""
import pytest

# test of tests/test_adapters_gpu.py or test_adapters_tiles_gpu.py: (rows, adapters) for few rows, (rows, adapters) in tiles
CASES = {
    "test_mixed_rows": ([(1, 8), (100, 7), (128, 1), (129, 9), (255, 300)], [(257, 12), (300, 4), (513, 513), (700, 6), (1500, 900)]),
    "test_requests_in_any_order": ([(64, 6)], [(130, 6), (513, 6)]),
    "test_a_broken_adapter_stays_with_its_rows": ([(3, 3), (40, 3)], [(300, 3), (600, 3), (1500, 4), (513, 30)]),
    "test_many_rows_of_one_tile": ([(112, 40), (256, 40), (250, 40), (500, 40)], []),
    "test_every_rank_and_every_adapter_counts": ([(4, 5)], [(300, 5)]),
    "test_offsets_beyond_32_bits": ([(5, 160), (300, 160)], [(513, 160), (600, 160)]),
    "test_every_adapter_broken_but_one": ([], [(700, 12)]),
    "test_captured_and_replayed_beside_eager_calls": ([(6, 9)], [(500, 9), (3000, 9)]),
    "test_two_threads_on_one_stream": ([(64, 9)], [(600, 9), (1100, 5)]),
}


@pytest.mark.parametrize("name", CASES)
def test_both_kernels_keep_their_tests(cuda_lib, name):
    few, tiles = CASES[name]
    assert [c for c in few if cuda_lib.fp4ar_adapters_few_rows(*c) != 1] == []
    assert [c for c in tiles if cuda_lib.fp4ar_adapters_few_rows(*c) != 0] == []


def test_bad_arguments(cuda_lib):
    assert cuda_lib.fp4ar_adapters_few_rows(-1, 1) == -1 and cuda_lib.fp4ar_adapters_few_rows(1, 0) == -1
    assert cuda_lib.fp4ar_adapters_few_rows(0, 1) == 1
