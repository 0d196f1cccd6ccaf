#!/bin/bash
# Build tuning variants of libnvk_paged_attn.so into build/variants/<name>.so: the library's own build (sources and flags of the
# Makefile) with more flags
# usage: tools/build_variants.sh name1:"-DNVK_X=1 -DNVK_Y=2" name2:"..."
# Select one at run time with NVK_LIB_PATH=build/variants/<name>.so
set -e
cd "$(dirname "$0")/.."
for spec in "$@"; do
  name="${spec%%:*}"; flags="${spec#*:}"
  [ "$name" = "$spec" ] && flags=
  make -s -j8 lib LIB="build/variants/$name.so" OBJ="build/variants/obj_$name" EXTRA="$flags"
  echo "built $name [$flags]"
done
