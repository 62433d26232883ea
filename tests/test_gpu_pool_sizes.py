"""Compactions and frees of pools around 2^18 pages, where the one-launch form's LDS passes 64 KB."""
import pytest

import test_gpu_pages

pytestmark = pytest.mark.gpu
check = test_gpu_pages.test_large_pools


@pytest.mark.parametrize("pages", [261887, 261888, 261889, 262144, 262145, 524287])
def test_pools_around_64_kilobytes_of_lds(ext, gpu, pages):
    check(ext, gpu, pages)
