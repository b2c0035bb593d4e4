// The output layer with its loss; declared in origin/functional.h.
#pragma once
#include "origin/functional.h"
