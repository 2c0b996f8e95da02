// Forwarding header: ccglib::orthogonalize::Orthogonalize is defined in <ccglib/b200_api.hpp>.
#pragma once
#include <ccglib/b200_api.hpp>
