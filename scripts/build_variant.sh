#!/bin/bash
# Builds a variant of libgsplat_hip.so for A/B measurements:  scripts/build_variant.sh <name> <extra hipcc flags>
#   -> opensplat_amd/csrc/libgsplat_hip_<name>.so ; run with GSPLAT_HIP_LIB=<that path> python bench.py ...
set -e
cd "$(dirname "$0")/.."
python3 -c "import sys; from opensplat_amd import _build; print('built', _build.build_variant(sys.argv[1], sys.argv[2:]))" "$@"
