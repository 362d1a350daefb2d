#!/bin/bash
# Variant of the library that differs in ONE kernel source's build flags (the other objects are reused):
#   tools/build_variant.sh <name> <a kernel file's name, as eval_f32> [extra hipcc flags...]  ->  build/variants/libbf_<name>.so
# Load it with BATCHFIRST_LIB=build/variants/libbf_<name>.so (batch_first_amd/_lib.py), tools/ab_time.py or tools/stamps.py.
set -e
name=$1; src=$2; shift 2
root=$(cd "$(dirname "$0")/.." && pwd)
obj="$root/build/variants/obj_$name"
mkdir -p "$obj"
cd "$obj"
# flags and objects as the Makefile has them
csrc="$root/batch_first_amd/csrc"
/opt/rocm/bin/hipcc $(make -s -C "$csrc" "flags-$src.o") "$@" --save-temps \
    -c "$root/batch_first_amd/csrc/$src.hip" -o $src.o
python3 "$root/tools/isa_hazards.py" $src-hip-amdgcn-amd-amdhsa-gfx950.s
grep "vgpr_spill_count\|\.vgpr_count\|\.agpr_count" $src-hip-amdgcn-amd-amdhsa-gfx950.s | head -9 || true
cd "$csrc"
objs=""
for o in $(make -s objects); do
    if [ "$o" = "$src.o" ]; then objs="$objs $obj/$o"; else objs="$objs $o"; fi
done
/opt/rocm/bin/hipcc -shared -fPIC --offload-arch=gfx950 $objs -o "$root/build/variants/libbf_$name.so"
rm -f "$obj"/*.hipi "$obj"/*.bc
echo "built build/variants/libbf_$name.so"
