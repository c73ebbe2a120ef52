"""The linear layer's kernel for few tokens and wide outputs, planned without a GPU (sgemm_i8.cpp against the stand-in of
test_i8_host.py): the plan has to be one that measurements bear out."""
import pytest

from test_i8_host import last, lib, linear  # noqa: F401

# (tokens, channels, features): microseconds on one B200 of "half" (CTA pairs on 256 x 128 tiles) and of the few-token kernel in 1, 2, 4 and 8 parts;
# captured graphs of calls over weights that together exceed L2, BF16 results
MEASURED = {
    (1, 4096, 4096): (9.8, 9.4, 7.6, 6.6, 6.6), (32, 4096, 4096): (10.0, 9.9, 8.9, 7.6, 7.7), (100, 4096, 4096): (10.0, 12.6, 12.3, 10.1, 22.2),
    (1, 8192, 4096): (12.3, 9.9, 9.3, 9.3, 12.9), (64, 8192, 4096): (10.8, 12.5, 12.9, 11.1, 17.8),
    (1, 12288, 4096): (15.1, 11.7, 12.7, 15.5, 18.4), (64, 12288, 4096): (13.1, 13.9, 15.5, 19.5, 25.8),
    (1, 14336, 4096): (15.3, 12.7, 14.2, 16.6, 22.6), (16, 14336, 4096): (14.3, 12.8, 14.4, 17.2, 23.7), (64, 14336, 4096): (14.0, 14.9, 16.5, 20.5, 31.3),
    (1, 4096, 14336): (24.5, 26.4, 16.3, 13.5, 13.5), (128, 4096, 14336): (24.3, 31.6, 23.1, 17.3, 32.2),
    (1, 28672, 4096): (25.6, 22.2, 25.8, 30.8, 40.3), (64, 28672, 4096): (24.4, 23.1, 32.7, 39.0, 57.0), (128, 28672, 4096): (25.4, 30.7, 56.3, 69.2, 123.8),
    (1, 28672, 8192): (47.7, 41.5, 42.5, 48.7, 55.0), (16, 28672, 8192): (44.6, 42.7, 44.4, 50.5, 58.4), (64, 28672, 8192): (45.7, 44.6, 51.0, 59.0, 71.7),
    (1, 8192, 28672): (53.2, 52.0, 42.5, 41.0, 43.9), (64, 8192, 28672): (49.9, 69.3, 49.5, 43.8, 50.1),
    (1, 32000, 4096): (27.5, 23.9, 27.5, 32.9, 45.0), (64, 32000, 4096): (26.1, 24.9, 34.2, 41.4, 62.8),
    (1, 57344, 8192): (84.0, 74.6, 81.9, 85.5, 101.2), (64, 57344, 8192): (88.7, 81.8, 97.8, 104.8, 135.9), (128, 57344, 8192): (90.9, 108.7, 135.4, 172.0, 280.5),
    (1, 128256, 4096): (94.0, 82.4, 95.5, 116.3, 175.4), (16, 128256, 4096): (87.9, 83.5, 97.1, 115.0, 176.9), (32, 128256, 4096): (84.0, 85.5, 105.1, 123.8, 192.6),
    (1, 151936, 2048): (58.4, 55.1, 71.8, 98.6, 181.1), (32, 151936, 2048): (59.1, 57.2, 78.8, 109.1, 202.9), (128, 151936, 2048): (59.3, 83.8, 189.4, 300.4, 589.8),
}


@pytest.mark.parametrize("tokens, channels, features", MEASURED)
def test_the_planned_kernel_is_near_the_fastest(lib, tokens, channels, features):   # noqa: F811
    assert linear(lib, lib.seam_handle(1, 0, 0), m=channels, n=tokens, k=features) == 0
    rec, times = last(lib), MEASURED[tokens, channels, features]
    name = lib.seam_name(rec.function).decode()
    time = times[0] if name == "i8_linear_half" else times[(1, 2, 4, 8).index(rec.parts) + 1]
    assert name != "generated_gemm" and time <= 1.06 * min(times), (name, rec.parts)


def test_no_estimate_lies_below_the_trip_from_memory(lib):   # noqa: F811
    """One token is bound by the weights wherever there are many: no tiles of 128 tokens there."""
    for channels in (12288, 14336, 28672, 57344, 128256, 151936):
        for features in (2048, 4096, 8192):
            assert linear(lib, lib.seam_handle(1, 0, 0), m=channels, n=1, k=features) == 0
            assert lib.seam_name(last(lib).function) == b"i8_linear_few_16"
