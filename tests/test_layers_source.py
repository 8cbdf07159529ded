"""Programs that use the layers' header: what compiled against it compiles still."""
import subprocess

import pytest

import c4s

SCALES = """
float scales(const c4s_kv_cache* cache) {   /* 8-bit codes' scales, as a program reads and sets them */
  float* k = cache->k_scale;
  float* v = cache->v_scale;
  return k[0] + v[1] + cache->k_scale[2];
}
void set(c4s_kv_cache* cache, float* k, float* v) { cache->k_scale = k; cache->v_scale = v; }
void set4(c4s_kv_cache* cache, uint8_t* k, uint8_t* v) { cache->k_scale = (float*)k; cache->v_scale = (float*)v; }
"""


@pytest.mark.parametrize("compiler", [["gcc", "-std=c11", "-x", "c"], ["g++", "-std=c++11", "-x", "c++"]])
def test_scales_are_floats(tmp_path, compiler):
    src = tmp_path / "scales.c"
    src.write_text(f'#include "{c4s.BATCH_HEADER}"\n' + SCALES)
    subprocess.run([*compiler, "-Wall", "-Wextra", "-Werror", "-fsyntax-only", str(src)], check=True)
